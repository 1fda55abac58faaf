"""The paged cache, prompt and tree attention together: speculative decoding."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _run(dtype, **kw):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from examples.speculative_paged import run
    return run(dtype, **kw)


@pytest.mark.parametrize("seed", [0, 1])
def test_speculative_equals_greedy(seed):
    out, plain, mean = _run(torch.float32, steps=10, seed=seed)
    for o, p in zip(out, plain):
        assert o == p[:len(o)] and len(o) >= 11
    for a, b in zip(out[:3], out[3:]):  # forks continue alike
        assert b == a[:len(b)]
    assert mean > 1.0  # some drafted tokens were accepted


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_speculative_16_bit_runs(dtype):
    out, plain, mean = _run(dtype, steps=6)
    assert all(len(o) >= 6 for o in out) and 1.0 <= mean <= 4.0
