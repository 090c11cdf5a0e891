"""lora_linear and its backward where numbers are hardest: ranks of unlike magnitude, infinities, the batch a token comes in, and
in-place results that autograd has seen."""
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


def _kinds(got, want, what):
    """The same entries are not a number, infinite and of either sign."""
    got, want = got.double().cpu(), want.double()
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        wrong = kind(got) != kind(want)
        assert not wrong.any(), f"{what}: {kind.__name__} in {wrong.nonzero()[:4].tolist()}, {int(wrong.sum())} entries"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 700])
@pytest.mark.parametrize("h, o", [(72, 136), (75, 139), (5, 6), (300, 600)])
@pytest.mark.parametrize("r", [1, 8, 12, 24, 64, 72, 128])
def test_infinities_of_the_definition(sampler, dtype, n, h, o, r):
    """An infinity anywhere gives what the definition has there: infinities of its sign, or no number where two meet or one
    meets a zero; fp64 says which.  Several come one at a time, since two in one sum mostly cancel to no number."""
    inf = float("inf")
    clean = _inputs(n, h, o, r, 2, dtype, seed=n + h + r, ids=torch.arange(n) % 3 - 1)
    last = int((clean["ids"] == 0).nonzero()[-1])             # the last token of adapter 0, which may fill up a tile
    places = [("hidden", (1, 0), inf), ("hidden", (last, h - 1), -inf), ("a", (0, 0, 0), inf), ("a", (0, r - 1, h - 1), -inf),
              ("b", (0, 0, 0), inf), ("b", (0, o - 1, r - 1), -inf), ("dy", (1, 0), inf), ("dy", (last, o - 1), -inf), ("dy", (last, 3), inf),
              ("base", (1, 2), -inf), ("dx", (1, 2), inf)]
    for name, at, value in places:
        c = dict(clean, **{name: clean[name].clone()})
        c[name][at] = value
        d = {k: v.cuda() for k, v in c.items()}
        out, u = sampler.lora_linear(d["base"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"], return_shrunk=True)
        want, want_u, _, _ = lora_ref.forward(c["base"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])
        _kinds(u, want_u, f"{name}{at}: shrunk")
        _kinds(out, want, f"{name}{at}: out")
        got = sampler.lora_linear_backward(d["dy"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"], u, d["dx"])
        want, _ = lora_ref.backward(c["dy"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"], u.cpu(), c["dx"])
        for x, w, what in zip(got, want, ("dhidden", "dlora_a", "dlora_b")):
            _kinds(x, w, f"{name}{at}: {what}")


@pytest.mark.parametrize("n", [3, 600])
@pytest.mark.parametrize("r", [1, 40])
def test_infinities_beside_the_smallest_numbers(sampler, n, r):
    """An infinity times the smallest fp16 numbers is one all the same."""
    tiny, inf = 2.0 ** -24, float("inf")
    full = lambda v, *shape: torch.full(shape, v, dtype=torch.float16)  # noqa: E731
    c = dict(base=full(0.0, n, 24), hidden=full(3 * tiny, n, 16), a=full(-tiny, 1, r, 16), b=full(5 * tiny, 1, 24, r),
             ids=torch.zeros(n, dtype=torch.int64), scaling=torch.ones(1), dy=full(-7 * tiny, n, 24))
    for name in ("hidden", "dy", "a", "b"):
        x = dict(c, **{name: c[name].clone()})
        x[name].view(-1)[1] = inf
        d = {k: v.cuda() for k, v in x.items()}
        out, u = sampler.lora_linear(d["base"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"], return_shrunk=True)
        want, want_u, _, _ = lora_ref.forward(x["base"], x["hidden"], x["a"], x["b"], x["ids"], x["scaling"])
        _kinds(u, want_u, f"{name}: shrunk")
        _kinds(out, want, f"{name}: out")
        got = sampler.lora_linear_backward(d["dy"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"], u)
        want, _ = lora_ref.backward(x["dy"], x["hidden"], x["a"], x["b"], x["ids"], x["scaling"], u.cpu(), None)
        for y, w, what in zip(got, want, ("dhidden", "dlora_a", "dlora_b")):
            _kinds(y, w, f"{name}: {what}")


def test_infinities_in_front_of_a_wide_output(sampler):
    """The same in the blocks of 1024 outputs, of which the last is cut short."""
    n, h, o, r, s, inf = 4100, 72, 65560, 11, 2, float("inf")
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda std, *shape: (torch.randn(*shape, generator=g, device="cuda") * std).bfloat16()  # noqa: E731
    dy, hidden, a, b = rnd(0.1, n, o), rnd(1.0, n, h), rnd(0.1, s, r, h), rnd(0.3, s, o, r)
    ids = torch.arange(n, device="cuda") % 3 - 1
    u = torch.randn(n, r, generator=g, device="cuda")
    scaling = torch.ones(s, device="cuda")
    dy[1, 65536], dy[4, 0], dy[4099, 65559], dy[2, 7] = inf, -inf, inf, -inf
    got = sampler.lora_linear_backward(dy, hidden, a, b, ids, scaling, u)
    with torch.device("cuda"):
        want, _ = lora_ref.backward(dy, hidden, a, b, ids, scaling, u, None)
    for x, w, what in zip(got, want, ("dhidden", "dlora_a", "dlora_b")):
        _kinds(x, w.cpu(), what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 3, 40])
def test_gradients_of_the_smallest_numbers(sampler, dtype, n):
    """dy and hidden of a few steps of fp16's smallest number, one token or a few: every product counts to its last bit."""
    c = _inputs(n, 72, 136, 12, 2, dtype, seed=n, ids=torch.arange(n) % 2)
    g = torch.Generator().manual_seed(n)
    for name in ("dy", "hidden"):
        c[name] = (torch.randint(-40, 41, c[name].shape, generator=g) * 2.0 ** -24).to(dtype)
    u = torch.randn(n, 12, generator=g)
    d = {k: v.cuda() for k, v in c.items()}
    got = sampler.lora_linear_backward(d["dy"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"], u.cuda(), d["dx"])
    want, bound = lora_ref.backward(c["dy"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"], u, c["dx"])
    for x, w, e, what in zip(got, want, bound, ("dhidden", "dlora_a", "dlora_b")):
        _within(x, w, e, what)


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


def test_in_place_is_seen_by_autograd(sampler):
    """A base that autograd has saved must not be overwritten unseen: the backward refuses it, as after torch's own in-place operators."""
    c = {k: v.cuda() for k, v in _inputs(9, 24, 40, 8, 2, torch.bfloat16, seed=2).items()}
    args = (c["hidden"], c["a"], c["b"], c["ids"])
    weight = torch.randn(40, 24, device="cuda").bfloat16().requires_grad_()
    base = torch.nn.functional.linear(c["hidden"], weight)
    loss = base.square().sum()                                # saves base
    before = base._version
    assert sampler.lora_linear(base, *args, inplace=True) is base
    assert base._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # rows of a larger tensor share its version; inference tensors have none
    store = torch.zeros(9, 64, device="cuda", dtype=torch.bfloat16)
    before = store._version
    sampler.lora_linear(store[:, 8:48], *args, inplace=True)
    assert store._version > before
    with torch.inference_mode():
        inside = c["base"].clone()
        sampler.lora_linear(inside, *args, inplace=True)
    assert torch.equal(inside, sampler.lora_linear(c["base"], *args))
    before = base._version
    sampler.lora_linear(base, *args)                          # out of place: nothing to see
    assert base._version == before
