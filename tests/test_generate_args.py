"""What Qwen2Runner.generate refuses before it touches its cache or runs the prompt (no GPU)."""
import pytest
import torch

from nanoserve_amd.qwen import Qwen2Runner, Qwen2Shape


@pytest.fixture
def runner(monkeypatch):
    r = Qwen2Runner.__new__(Qwen2Runner)
    r.shape = Qwen2Shape(layers=1, hidden=512, heads=4, kv_heads=2, intermediate=1024, vocab=2000)
    r.dev, r.logits = torch.device("cpu"), torch.zeros(1, 2000, dtype=torch.bfloat16)

    class _Kernels:
        def sample_workspace(self, *args, **kw):
            return torch.zeros(16, dtype=torch.uint8)

    def run(*args, **kw):
        raise AssertionError("the prompt was run")

    r.k = _Kernels()
    monkeypatch.setattr(Qwen2Runner, "alloc_cache", run)
    return r


@pytest.mark.parametrize("kw,err", [
    (dict(temperature=-0.1), ValueError), (dict(temperature=float("nan")), ValueError),
    (dict(temperature=0.7, top_k=-1), ValueError), (dict(temperature=0.7, top_p=1.5), ValueError),
    (dict(temperature=0.7, top_p=float("nan")), ValueError), (dict(temperature=0.7, min_p=-0.5), ValueError),
    (dict(temperature=0.7, min_p=2), ValueError), (dict(temperature=0.7, u=torch.zeros(2)), ValueError),
    (dict(temperature=0.7, u=torch.zeros(3, 1)), ValueError),
    (dict(temperature=0.7, u=torch.zeros(3, device="meta")), ValueError),
    (dict(temperature=0.7, u=torch.zeros(3, dtype=torch.float64)), TypeError),
    (dict(temperature=0.7, u=[0.1, 0.2, 0.3]), TypeError)], ids=str)
def test_generate_refuses_before_the_prompt(runner, kw, err):
    with pytest.raises(err):
        runner.generate(torch.arange(5), 3, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.0, top_k=-1, top_p=3.0), dict(temperature=0.7, u=torch.zeros(3)),
                                dict(temperature=0.7, top_k=5, top_p=0.5, min_p=1)], ids=str)
def test_generate_runs_the_prompt(runner, kw):
    with pytest.raises(AssertionError, match="was run"):
        runner.generate(torch.arange(5), 3, **kw)
