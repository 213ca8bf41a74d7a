"""The C++ binding of attention_shared and verify_drafts: it takes what the Python entry points take, gives the same bits and the same counts
of launches as the way through ctypes, and leaves everything else to the checks there."""
import pytest
import torch

from hipinfer_b200.kernels import drafts, library, ops


def test_what_it_does_not_take_is_left_to_the_checks():
    module = library.load_binding("drafts")
    if module is None:
        pytest.skip("no host compiler or no headers: operations go through ctypes")
    assert module.attend(None, 1, "x", [], 0, None, None, 0) is None and module.verify(*[None] * 8) is None
    cpu = torch.zeros(2, 2)
    assert module.attend(cpu, cpu, cpu, cpu, 0, None, None, 0) is None and module.verify(*[cpu] * 7, None) is None
    for call, n in ((module.attend, 7), (module.verify, 9), (module.bind, 2)):
        with pytest.raises(TypeError):
            call(*[None] * n)


def attend_args(dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    plan = ops.SharedPlan([1, 3, 2], [70, 90, 81], [(0, 3, 64)], 8, 2, 64, 16, dtype)
    q = torch.randn(6, 8 * 64, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(20, 2, 16, 64, generator=g, device="cuda").to(dtype) for _ in range(2))
    table = torch.tensor([[0, 1, 2, 3, 4, -1], [0, 1, 2, 3, 5, 6], [0, 1, 2, 3, 7, 8]], dtype=torch.int32, device="cuda")
    return dict(q=q, k_cache=k, v_cache=v, block_table=table, plan=plan)


def verify_args(K=3, probs=None):
    g = torch.Generator(device="cuda").manual_seed(2)
    R, V = 4, 1003
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    p = None if probs is None else torch.softmax(torch.randn(R, K, V, generator=g, device="cuda"), -1).to(probs)
    return dict(logits=torch.randn(R * (K + 1), V, generator=g, device="cuda") * 2, start=t(*[r * (K + 1) for r in range(R)]),
                n_drafts=t(*[min(r, K) for r in range(R)]), drafts=torch.randint(V, (R, K), generator=g, device="cuda", dtype=torch.int32),
                temperature=torch.tensor([0.0, 0.7, 1.0, 1.3], device="cuda"), uniform=torch.rand(R, K, generator=g, device="cuda"),
                noise=torch.empty(R, V, device="cuda").exponential_(generator=g), draft_probs=p)


def both(monkeypatch, call):
    """call() through the binding, then through ctypes, with the launches of each."""
    if library.load_binding("drafts") is None:
        pytest.skip("no host compiler or no headers: operations go through ctypes")
    call()
    assert drafts._bound
    out = []
    for bound in (drafts._bound, False):
        with monkeypatch.context() as m:
            m.setattr(drafts, "_bound", bound)
            before = library.launches[0]
            out.append((call(), library.launches[0] - before))
    torch.cuda.synchronize()
    ops.check_device_status()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_has_the_same_bits(monkeypatch, dtype):
    a = attend_args(dtype)
    (x, n), (y, m) = both(monkeypatch, lambda: ops.attention_shared(**a))
    assert torch.equal(x, y) and x.dtype == dtype and x.shape == (6, 512) and x.is_contiguous() and n == m == 2
    wide = torch.zeros(6, 700, dtype=dtype, device="cuda")
    wide[:, 100:612] = a["q"]
    given = torch.empty(6, 512, dtype=dtype, device="cuda")
    (x, _), (y, _) = both(monkeypatch, lambda: ops.attention_shared(**{**a, "q": wide[:, 100:612]}, out=given, scale=0.3).clone())
    assert torch.equal(x, y) and torch.equal(given, y)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        (x, _), (y, _) = both(monkeypatch, lambda: ops.attention_shared(**a))
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("K, probs", [(3, None), (3, torch.float32), (2, torch.bfloat16), (0, None), (0, torch.float32)])
def test_verification_has_the_same_bits(monkeypatch, K, probs):
    a = verify_args(K, probs)
    (x, n), (y, m) = both(monkeypatch, lambda: ops.verify_drafts(**a))
    assert n == m == 2
    for s, t in zip(x, y):
        assert torch.equal(s, t) and s.dtype == t.dtype and s.shape == t.shape and s.is_contiguous()


@pytest.mark.gpu
def test_refusals_say_what_is_wrong():
    a = attend_args(torch.bfloat16)
    for bad, words in ((dict(q=a["q"][:5]), "6 rows"), (dict(q=a["q"].float()), "bfloat16"), (dict(k_cache=a["k_cache"][:, :1]), "keys"),
                       (dict(v_cache=a["v_cache"].float()), "values"), (dict(block_table=a["block_table"].long()), "block table"),
                       (dict(block_table=a["block_table"][:, :5]), "block table"), (dict(out=a["q"].float()), "out"), (dict(block_table=a["block_table"].cpu()), "CUDA")):
        with pytest.raises(ops.KernelError, match=words):
            ops.attention_shared(**{**a, **bad})
    v = verify_args()
    for bad, words in ((dict(noise=v["noise"][:, 1:]), "noise"), (dict(start=v["start"].long()), "start"), (dict(drafts=v["drafts"].t()), "n_drafts|start|drafts"),
                       (dict(logits=v["logits"].half()), "float16"), (dict(uniform=v["uniform"].cpu()), "CUDA"),
                       (dict(draft_probs=torch.zeros(4, 2, 1003, device="cuda")), "draft_probs")):
        with pytest.raises(ops.KernelError, match=words):
            ops.verify_drafts(**{**v, **bad})
    torch.cuda.synchronize()
    ops.check_device_status()
