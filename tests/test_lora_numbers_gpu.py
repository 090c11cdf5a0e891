"""lora_linear and its backward where numbers are hardest: ranks of unlike magnitude, and the batch a token comes in."""
import pytest
import torch

from oracle import lora_ref
from tests.test_lora_gpu import _inputs, _within

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, h", [(20, 72), (20, 2100), (700, 72), (700, 2100)])
@pytest.mark.parametrize("r", [2, 12, 24, 64, 128])
def test_ranks_of_unlike_magnitude(sampler, dtype, n, h, r):
    """Rows of A over a range of 2^20, columns of B the other way round: every rank matters as much as the others, and each is
    held to its own bound (2^-17 of |u_r| |B_r|), the smallest u beside the largest."""
    c = _inputs(n, h, 136, r, 3, dtype, seed=n + h + r)
    by = (2.0 ** torch.linspace(10, -10, r).round())
    c["a"] = (c["a"].float() * by[:, None]).to(dtype)
    c["b"] = (c["b"].float() / by).to(dtype)
    d = {k: v.cuda() for k, v in c.items()}
    out, u = sampler.lora_linear(d["base"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"], return_shrunk=True)
    y, want_u, ey, eu = lora_ref.forward(c["base"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])
    _within(u, want_u, eu, "shrunk")
    _within(out, y, ey, "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 600])
def test_a_small_rank_alone_in_a_column(sampler, dtype, n):
    """u = (100, 3e-6) and a column of B that is (0, 30000): the result is the small rank's alone."""
    a = torch.zeros(1, 2, 8)
    a[0, 0, 0], a[0, 1, 0] = 100.0, 3.1e-6
    b = torch.zeros(1, 16, 2)
    b[0, :, 1] = 30000.0
    hidden = torch.zeros(n, 8)
    hidden[:, 0] = 1.0
    c = [t.to(dtype) for t in (torch.zeros(n, 16), hidden, a, b)] + [torch.zeros(n, dtype=torch.int64)]
    y, _, bound, _ = lora_ref.forward(*c, torch.ones(1))
    _within(sampler.lora_linear(*[t.cuda() for t in c]), y, bound, "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r, h", [(16, 72), (16, 2100), (24, 2100), (64, 1500), (128, 2100)])
def test_bits_of_a_token_whatever_the_batch(sampler, dtype, r, h):
    """Both routes of few and many tokens (n R <= 8192 and n <= 512, or not), and both ways of adding the segments of H (fewer
    than 512 tiles, or not), give a token the same bits."""
    c = {k: v.cuda() for k, v in _inputs(20000, h, 72, r, 3, dtype, seed=5 + r).items()}
    call = lambda i: sampler.lora_linear(c["base"][i], c["hidden"][i], c["a"], c["b"], c["ids"][i], c["scaling"], return_shrunk=True)  # noqa: E731
    whole = call(slice(None))
    few = 8192 // r
    for i in (slice(0, 1), slice(777, 777 + min(few, 512)), slice(777, 778 + min(few, 512)), slice(3000, 3513), slice(1000, 1000 + 16200),
              slice(19999, 20000), torch.tensor([5, 19000, 64, 3], device="cuda")):
        part = call(i)
        assert torch.equal(part[0], whole[0][i]) and torch.equal(part[1], whole[1][i])
