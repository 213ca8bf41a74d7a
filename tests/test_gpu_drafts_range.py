"""Verification of drafted tokens over the whole range of temperatures and finite logits, against the same 64-bit decisions as elsewhere."""
import math

import pytest
import torch

from hipinfer_b200.kernels import ops
from test_gpu_drafts import BF16, DEV, F32, check_verify, fixed, make_verify

pytestmark = pytest.mark.gpu
LOWEST = {F32: torch.finfo(F32).min, BF16: torch.finfo(BF16).min}


@pytest.mark.parametrize("t", [1e-3, 1e-6, 1e-7, 1e-8, 1e-9, 1e-10, 1e-12, 1e-20, 1e-37, 1e-45, 1e6, 1e30, math.inf])
@pytest.mark.parametrize("dtype,probs", [(F32, None), (F32, F32), (BF16, BF16), (BF16, None)])
def test_any_temperature_above_zero(t, dtype, probs):
    """Nearly greedy and nearly uniform draws: the largest logit has exponent 0 whatever it is multiplied by. (At the small ones the distribution is a
    point, or some points where logits are alike, as 16-bit ones are.)"""
    logits, start, lens, drafts, _, u, noise, q = make_verify(40, 3, 1003, dtype, probs, seed=5, greedy=0)
    best = logits[torch.tensor(start, device=DEV)].float().argmax(-1).to(torch.int32)
    drafts[::2, 0] = best[::2]                    # half of the first drafts are the likeliest token
    check_verify(logits, start, lens, drafts, torch.full((40,), t, device=DEV), u, noise, q, allow=0.1)


@pytest.mark.parametrize("V", [5, 700, 40001])
@pytest.mark.parametrize("t", [1e-8, 1e-3, 0.7, 1.0, 30.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_lowest_finite_number_as_a_mask(dtype, t, V):
    """Rows of nothing else are uniform; beside other logits such a one weighs nothing."""
    logits, start, lens, drafts, _, u, noise, _ = make_verify(12, 2, V, dtype, seed=V, greedy=0)
    gen = torch.Generator(device=DEV).manual_seed(1)
    logits[torch.rand(logits.shape, generator=gen, device=DEV) < 0.6] = LOWEST[dtype]
    logits[::3] = LOWEST[dtype]
    check_verify(logits, start, lens, drafts, torch.full((12,), t, device=DEV), u, noise, allow=0.1)
    x = torch.full((1, V), LOWEST[dtype], dtype=dtype)
    token, count, logp = fixed(x.float().tolist(), t=t, noise=[1.0 + (v != V // 2) for v in range(V)])
    assert token == [V // 2] and count == 1 and abs(logp[0] + math.log(V)) <= 2.0 ** -24 * (64 + V)


def test_large_finite_logits():
    top = torch.finfo(F32).max
    for t in (0.0, 1e-3, 1.0):
        assert fixed([[3e38, top, -top, 0.0]], t=t) == [[1], 1, [0.0]]
        assert fixed([[-3e38, -top, -3e38]], t=t, noise=[1.0, 1e-9, 0.5])[:2] == [[0 if t == 0 else 2], 1]
        # a draft that is the largest, and one that is not
        assert fixed([[1.0, top, 3.2e38], [0.0, 2.5e38, top]], n=1, t=t, drafts=[1], u=[0.99]) == [[1, 2], 2, [0.0, 0.0]]
        assert fixed([[1.0, top, 3.2e38], [0.0, 2.5e38, top]], n=1, t=t, drafts=[2], u=[0.01]) == [[1, -1], 1, [0.0, 0.0]]
    assert fixed([[-3e38, -top, -3e38]], t=1.0)[2][0] == pytest.approx(-math.log(2), rel=1e-6)


def test_requests_at_different_temperatures_in_one_call():
    logits, start, lens, drafts, _, u, noise, _ = make_verify(30, 2, 3001, seed=8, greedy=0)
    t = torch.tensor([0.0, 1e-9, 0.8, 1e-38, 5.0] * 6, device=DEV)
    check_verify(logits, start, lens, drafts, t, u, noise, allow=0.1)
    ops.check_device_status()
