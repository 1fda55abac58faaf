"""What new-token attention writes is there for the kernel that comes next on the
stream, and a row tile's shared memory holds what was copied for it."""
import pytest
import torch

from adakv_b200.attention import AdaKVCache, adakv_decode_attention
from adakv_b200.prompt import prompt_attention
from tests.extend_cases import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def rnd(*shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_reads_a_short_prompts_output(dtype, D):
    """The sparse decode's kernels read their query before they wait for the kernel
    in front of them: here the attention of a prompt short enough to be one launch."""
    cache = AdaKVCache(16)
    cache.append_prefill(rnd(8, 3000, D, seed=1, dtype=dtype), rnd(8, 3000, D, seed=2, dtype=dtype))
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    k, v = rnd(40, 8, D, seed=3, dtype=dtype), rnd(40, 8, D, seed=4, dtype=dtype)
    qs = [rnd(40, 32, D, seed=10 + i, dtype=dtype) for i in range(6)]
    out = torch.zeros((40, 32, D), dtype=dtype, device="cuda")
    want = []
    for q in qs:
        prompt_attention(q, k, v, cu, out=out)
        torch.cuda.synchronize()
        want.append(adakv_decode_attention(out[39].clone(), cache, 32))
        torch.cuda.synchronize()
    got = []
    for q in qs * 5:
        prompt_attention(q, k, v, cu, out=out)
        got.append(adakv_decode_attention(out[39], cache, 32))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 6])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,prefix", [([40] * 30, [0] * 30), ([3, 64, 65, 17, 1] * 6, [0] * 30), ([5] * 24, [9] * 24)])
def test_many_short_row_tiles_to_a_cta(D, new, prefix):
    """32-bit row tiles of one to three key tiles, several behind one another in each
    CTA: K of each comes into the same shared memory."""
    c = Case(new, prefix, 64, 16, D, torch.float32, seed=sum(new))
    d = c.device
    pages = c.pages() if sum(prefix) else None
    slots = c.slots.int().to(d) if pages else None
    first = None
    for _ in range(4):
        out, lse = prompt_attention(c.q.to(d), c.k.to(d), c.v.to(d), c.cu_tensor(), pages, slots=slots, return_lse=True)
        if first is None:
            first = out, lse
            c.check(out, lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
