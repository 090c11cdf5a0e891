"""lora_linear and its backward on the GPU against fp64, element by element within what rounding may do (oracle/lora_ref.py)."""
import pytest
import torch

from oracle import lora_ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _inputs(n, h, o, r, s, dtype, seed, ids=None):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda std, *shape: (torch.randn(*shape, generator=g) * std).to(dtype)  # noqa: E731
    if ids is None:
        ids = torch.randint(-1, s, (n,), generator=g)
    return dict(base=rnd(1.0, n, o), hidden=rnd(1.0, n, h), a=rnd(h ** -0.5, s, r, h), b=rnd(0.3, s, o, r), ids=ids,
                scaling=torch.rand(s, generator=g) + 0.5, dy=rnd(0.1, n, o), dx=rnd(0.5, n, h))


def _within(got, want, bound, what):
    dtype, got = got.dtype, got.cpu().double()
    assert got.shape == want.shape
    # a value beyond the type's range rounds to an infinity (fp16: from 65520 on); within its bound of that border it may do either
    limit = torch.finfo(dtype).max * (1.0 + torch.finfo(dtype).eps / 4)
    sure = want.abs() - bound >= limit
    assert torch.equal(got[sure], torch.sign(want[sure]) * float("inf")), f"{what}: a result beyond the range of {dtype}"
    near = (want.abs() + bound >= limit) & ~torch.isfinite(got) & (torch.sign(got) == torch.sign(want))
    got = torch.where(sure | near, want, got)
    over = ((got - want).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 0, f"{what}: {over} beyond its bound"


def _check(sampler, c, backward=True):
    d = {k: v.cuda() for k, v in c.items()}
    out, u = sampler.lora_linear(d["base"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"], return_shrunk=True)
    y, want_u, ey, eu = lora_ref.forward(c["base"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])
    assert out.dtype == c["base"].dtype and u.dtype == torch.float32
    _within(u, want_u, eu, "shrunk")
    _within(out, y, ey, "out")
    none = (c["ids"] < 0) | (c["ids"] >= c["a"].shape[0])
    assert torch.equal(out.cpu()[none], c["base"][none]) and not u.cpu()[none].any()
    if not backward:
        return out, u
    for dx_base in (c["dx"], None):
        got = sampler.lora_linear_backward(d["dy"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"], shrunk=u,
                                           dhidden_base=None if dx_base is None else d["dx"])
        want, bound = lora_ref.backward(c["dy"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"], u.cpu(), dx_base)
        for x, w, e, what in zip(got, want, bound, ("dhidden", "dlora_a", "dlora_b")):
            _within(x, w, e, what)
        assert got[0].dtype == c["hidden"].dtype and got[1].dtype == got[2].dtype == torch.float32
    again = sampler.lora_linear_backward(d["dy"], d["hidden"], d["a"], d["b"], d["ids"], d["scaling"])
    assert all(torch.equal(x, y) for x, y in zip(got, again))       # u computed again: the same bits
    return out, u


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 129, 700])
def test_token_counts(sampler, dtype, n):
    _check(sampler, _inputs(n, 136, 264, 16, 3, dtype, seed=n))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r", [1, 3, 8, 12, 16, 17, 24, 32, 40, 64, 65, 96, 127, 128])
def test_ranks(sampler, dtype, r):
    _check(sampler, _inputs(70, 192, 320, r, 2, dtype, seed=r))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h, o", [(1, 1), (7, 3), (8, 8), (33, 65), (64, 63), (255, 257), (1024, 1032), (1025, 100), (2056, 1000),
                                  (4096, 72)])
def test_widths(sampler, dtype, h, o):
    for r in (8, 20):
        _check(sampler, _inputs(37, h, o, r, 2, dtype, seed=h + o + r))


@pytest.mark.parametrize("s", [1, 2, 64, 1023])
def test_numbers_of_adapters(sampler, s):
    _check(sampler, _inputs(150, 64, 72, 8, s, torch.bfloat16, seed=s))


def test_orders_of_adapters(sampler):
    n, s = 333, 4
    for ids in (torch.full((n,), -1), torch.full((n,), 3), torch.arange(n) % s, torch.arange(n - 1, -1, -1) * s // n,
                torch.where(torch.arange(n) % 2 == 0, 5, 1), torch.full((n,), 1 << 40), torch.full((n,), -(1 << 40))):
        _check(sampler, _inputs(n, 72, 80, 16, s, torch.bfloat16, seed=1, ids=ids))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens(sampler, dtype):
    """More tokens than a tile of the backward holds, and enough tiles that one workgroup adds a token's segments itself."""
    c = _inputs(20000, 1096, 40, 8, 2, dtype, seed=2)
    _check(sampler, c)


@pytest.mark.parametrize("r", [16, 64])
def test_vocabulary_width(sampler, r):
    """The lm_head's width, every token its own adapter and all of one, with the wide blocks of the backward."""
    c = _inputs(33, 256, 128256, r, 33, torch.bfloat16, seed=3, ids=torch.randperm(33, generator=torch.Generator().manual_seed(1)))
    _check(sampler, c, backward=False)
    _check(sampler, _inputs(1100, 64, 32000 + 8, r, 1, torch.bfloat16, seed=4, ids=torch.zeros(1100, dtype=torch.int64)))


def test_result_of_a_token_does_not_depend_on_the_batch(sampler):
    c = {k: v.cuda() for k, v in _inputs(20000, 2100, 48, 16, 3, torch.bfloat16, seed=5).items()}
    call = lambda i: sampler.lora_linear(c["base"][i], c["hidden"][i], c["a"], c["b"], c["ids"][i], c["scaling"], return_shrunk=True)  # noqa: E731
    whole = call(slice(None))
    for i in (slice(0, 1), slice(777, 900), slice(19999, 20000), torch.tensor([5, 19000, 64, 3], device="cuda")):
        part = call(i)
        assert torch.equal(part[0], whole[0][i]) and torch.equal(part[1], whole[1][i])


def test_scaling_and_integer_types(sampler):
    c = {k: v.cuda() for k, v in _inputs(50, 64, 64, 8, 3, torch.float16, seed=6).items()}
    args = (c["base"], c["hidden"], c["a"], c["b"])
    want = sampler.lora_linear(*args, c["ids"], torch.full((3,), 0.75, device="cuda"))
    assert torch.equal(sampler.lora_linear(*args, c["ids"].to(torch.int32), 0.75), want)
    assert torch.equal(sampler.lora_linear(*args, c["ids"].cpu(), torch.full((3,), 0.75, dtype=torch.float64)), want)
    assert torch.equal(sampler.lora_linear(*args, c["ids"], 0.0), c["base"])


def test_layouts_and_in_place(sampler):
    g = torch.Generator().manual_seed(7)
    n, h, o, r, s = 60, 72, 136, 16, 3
    wide = lambda d, off: (torch.randn(n, d + 40, generator=g).bfloat16().cuda())[:, off:off + d]  # noqa: E731
    c = {k: v.cuda() for k, v in _inputs(n, h, o, r, s, torch.bfloat16, seed=8).items()}
    for off in (0, 8, 3):
        base, hidden, dy, dxb = wide(o, off), wide(h, off), wide(o, off), wide(h, off)
        out, u = sampler.lora_linear(base, hidden, c["a"], c["b"], c["ids"], c["scaling"], return_shrunk=True)
        want, want_u = sampler.lora_linear(base.contiguous(), hidden.contiguous(), c["a"], c["b"], c["ids"], c["scaling"],
                                           return_shrunk=True)
        assert torch.equal(out, want) and torch.equal(u, want_u)
        got = sampler.lora_linear_backward(dy, hidden, c["a"], c["b"], c["ids"], c["scaling"], u, dxb)
        ref = sampler.lora_linear_backward(dy.contiguous(), hidden.contiguous(), c["a"], c["b"], c["ids"], c["scaling"], u,
                                           dxb.contiguous())
        assert all(torch.equal(x, y) for x, y in zip(got, ref))
        # in place, on a view with gaps: what lies beside the rows stays as it was
        store = torch.randn(n, o + 40, generator=g).bfloat16().cuda()
        before = store.clone()
        store[:, off:off + o] = base
        assert sampler.lora_linear(store[:, off:off + o], hidden, c["a"], c["b"], c["ids"], c["scaling"], inplace=True).data_ptr() == \
            store[:, off:off + o].data_ptr()
        assert torch.equal(store[:, off:off + o], want)
        assert torch.equal(store[:, :off], before[:, :off]) and torch.equal(store[:, off + o:], before[:, off + o:])
    # [B, L, ..] and one token without a batch; transposed adapters
    b3 = c["base"].view(5, 12, o)
    got = sampler.lora_linear(b3, c["hidden"].view(5, 12, h), c["a"], c["b"], c["ids"].view(5, 12), c["scaling"])
    want = sampler.lora_linear(c["base"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])
    assert got.shape == (5, 12, o) and torch.equal(got.view(n, o), want)
    a_t, b_t = c["a"].transpose(1, 2).contiguous().transpose(1, 2), c["b"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(sampler.lora_linear(c["base"], c["hidden"], a_t, b_t, c["ids"], c["scaling"]), want)
    one = sampler.lora_linear(c["base"][4], c["hidden"][4], c["a"], c["b"], c["ids"][4], c["scaling"])
    assert one.shape == (o,) and torch.equal(one, want[4])
    with pytest.raises(ValueError, match="inplace"):
        sampler.lora_linear(c["base"].view(5, 12, o).transpose(0, 1), c["hidden"].view(12, 5, h), c["a"], c["b"],
                            c["ids"].view(12, 5), inplace=True)


def test_rows_that_lie_more_than_4_gib_apart(sampler):
    n, h, o, r, s = 70, 64, 72, 16, 2
    c = {k: v.cuda() for k, v in _inputs(n, h, o, r, s, torch.bfloat16, seed=12).items()}
    step = 1 << 25                                            # 64 MiB per row: 4.4 GiB in all
    store = torch.empty(n * step, dtype=torch.bfloat16, device="cuda")

    def far(t, at):
        v = store.as_strided(t.shape, (step, 1), at)
        v.copy_(t)
        return v

    base, hidden, dy, dx = far(c["base"], 0), far(c["hidden"], 1024), far(c["dy"], 2048), far(c["dx"], 4096)
    out, u = sampler.lora_linear(base, hidden, c["a"], c["b"], c["ids"], c["scaling"], return_shrunk=True)
    want, want_u = sampler.lora_linear(c["base"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"], return_shrunk=True)
    assert torch.equal(out, want) and torch.equal(u, want_u)
    got = sampler.lora_linear_backward(dy, hidden, c["a"], c["b"], c["ids"], c["scaling"], u, dx)
    ref = sampler.lora_linear_backward(c["dy"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"], u, c["dx"])
    assert all(torch.equal(x, y) for x, y in zip(got, ref))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_stay_with_their_token(sampler, dtype):
    c = {k: v.cuda() for k, v in _inputs(40, 64, 72, 16, 2, dtype, seed=9, ids=torch.arange(40) % 2).items()}
    want = sampler.lora_linear(c["base"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])
    dx = sampler.lora_linear_backward(c["dy"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])[0]
    hidden, base, dy = c["hidden"].clone(), c["base"].clone(), c["dy"].clone()
    hidden[3, 5], base[7, 11], hidden[9, 0], dy[12, 4] = float("inf"), float("nan"), float("nan"), float("-inf")
    got = sampler.lora_linear(base, hidden, c["a"], c["b"], c["ids"], c["scaling"])
    fine = torch.ones(40, dtype=torch.bool)
    fine[[3, 7, 9]] = False
    assert torch.equal(got[fine.cuda()], want[fine.cuda()])
    assert not torch.isfinite(got[3]).any() and not torch.isfinite(got[9]).any()
    assert torch.isnan(got[7, 11]) and torch.equal(torch.cat([got[7, :11], got[7, 12:]]), torch.cat([want[7, :11], want[7, 12:]]))
    gdx, da, db = sampler.lora_linear_backward(dy, c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])
    rows = torch.ones(40, dtype=torch.bool)
    rows[12] = False
    assert torch.equal(gdx[rows.cuda()], dx[rows.cuda()]) and not torch.isfinite(gdx[12]).any()
    assert torch.isfinite(da[1]).all() and torch.isfinite(db[1]).all()          # token 12 belongs to adapter 0
    assert not torch.isfinite(da[0]).any() and not torch.isfinite(db[0, 4]).any() and torch.isfinite(db[0, 5]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_and_large_values(sampler, dtype):
    """Gradients down to the smallest numbers of the type and products near its largest keep their relative precision."""
    for seed, (sx, sb, sd) in enumerate(((1.0, 0.3, 1e-6), (30.0, 100.0, 1e-3), (1e-3, 1e-3, 1.0))):
        c = _inputs(90, 128, 136, 16, 2, dtype, seed=seed)
        c["hidden"] = (c["hidden"].float() * sx).to(dtype)
        c["b"] = (c["b"].float() * sb / 0.3).to(dtype)
        c["dy"] = (c["dy"].float() * sd).to(dtype)
        c["base"], c["dx"] = torch.zeros_like(c["base"]), torch.zeros_like(c["dx"])
        _check(sampler, c)


def test_empty_calls(sampler):
    c = {k: v.cuda() for k, v in _inputs(4, 16, 24, 8, 2, torch.bfloat16, seed=1).items()}
    out, u = sampler.lora_linear(c["base"][:0], c["hidden"][:0], c["a"], c["b"], c["ids"][:0], return_shrunk=True)
    assert out.shape == (0, 24) and u.shape == (0, 8)
    dx, da, db = sampler.lora_linear_backward(c["dy"][:0], c["hidden"][:0], c["a"], c["b"], c["ids"][:0])
    assert dx.shape == (0, 16) and da.shape == (2, 8, 16) and db.shape == (2, 24, 8) and not da.any() and not db.any()


def test_graph_replay_and_two_streams(sampler):
    sets = [{k: v.cuda() for k, v in _inputs(200, 1100, 264, 16, 4, torch.bfloat16, seed=s).items()} for s in range(3)]

    def step(c):
        out, u = sampler.lora_linear(c["base"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"], return_shrunk=True)
        return (out, u) + sampler.lora_linear_backward(c["dy"], c["hidden"], c["a"], c["b"], c["ids"], c["scaling"], u, c["dx"])

    want = [step(c) for c in sets]
    buf = {k: v.clone() for k, v in sets[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    for i in (0, 1, 2, 1, 0):
        for k in buf:
            buf[k].copy_(sets[i][k])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = step(sets[(i + 1) % 3])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        assert all(torch.equal(a, b) for a, b in zip(other, want[(i + 1) % 3]))


def test_the_largest_number_of_tokens(sampler):
    """2^20 tokens: every tile list at its longest; a second call of the same tokens in another order gives every token the same bits."""
    n, h, o, r, s = 1 << 20, 8, 16, 4, 1023
    g = torch.Generator(device="cuda").manual_seed(21)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()  # noqa: E731
    base, hidden, a, b = rnd(n, o), rnd(n, h), rnd(s, r, h), rnd(s, o, r)
    ids = torch.randint(-1, s + 1, (n,), generator=g, device="cuda")
    out, u = sampler.lora_linear(base, hidden, a, b, ids, 0.5, return_shrunk=True)
    some = torch.randint(0, n, (4000,), generator=g, device="cuda")
    some[0], some[1] = 0, n - 1
    pick = lambda t: t[some].cpu()  # noqa: E731
    y, want_u, ey, eu = lora_ref.forward(pick(base), pick(hidden), a.cpu(), b.cpu(), pick(ids), torch.full((s,), 0.5))
    _within(out[some], y, ey, "out")
    _within(u[some], want_u, eu, "shrunk")
    order = torch.randperm(n, generator=g, device="cuda")
    assert torch.equal(sampler.lora_linear(base[order], hidden[order], a, b, ids[order], 0.5), out[order])
    dx, da, db = sampler.lora_linear_backward(base, hidden, a, b, ids, 0.5, u)
    got = [x.clone() for x in (da, db)]
    # an adapter's gradients are sums over its tokens alone: those of a few adapters, in fp64
    for i in (0, 511, 1022):
        mine = ids == i
        c = [t[mine].cpu() for t in (base, hidden, u)]
        want, bound = lora_ref.backward(c[0], c[1], a[i:i + 1].cpu(), b[i:i + 1].cpu(), torch.zeros(len(c[0]), dtype=torch.int64),
                                        torch.full((1,), 0.5), c[2], None)
        _within(dx[mine], want[0], bound[0], "dhidden")
        _within(got[0][i:i + 1], want[1], bound[1], "dlora_a")
        _within(got[1][i:i + 1], want[2], bound[2], "dlora_b")
    with pytest.raises(ValueError, match="tokens"):
        sampler.lora_linear(rnd(n + 1, 1), rnd(n + 1, 1), rnd(1, 1, 1), rnd(1, 1, 1), torch.zeros(n + 1, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 700])
@pytest.mark.parametrize("o", [136, 139])
def test_infinities_of_an_adapter_stay_with_its_tokens(sampler, dtype, n, o):
    """Adapter 0 diverged (infinities and NaN in both matrices): tokens of other adapters, and those without one, keep their results."""
    c = _inputs(n, 72, o, 12, 3, dtype, seed=n)
    c["ids"] = torch.arange(n) % 4 - 1
    d = {k: v.cuda() for k, v in c.items()}
    run = lambda a, b: (sampler.lora_linear(d["base"], d["hidden"], a, b, d["ids"], d["scaling"], return_shrunk=True))  # noqa: E731
    back = lambda a, b, u: sampler.lora_linear_backward(d["dy"], d["hidden"], a, b, d["ids"], d["scaling"], u, d["dx"])  # noqa: E731
    want, u = run(d["a"], d["b"])
    grads = back(d["a"], d["b"], u)
    a, b = d["a"].clone(), d["b"].clone()
    a[0, 0, :] = float("inf")
    a[0, :, 3] = float("nan")
    b[0, :, 0] = float("inf")
    b[0, 5, :] = float("nan")
    out, u_bad = run(a, b)
    bad = back(a, b, u_bad)
    others = d["ids"] != 0
    assert torch.equal(out[others], want[others]) and torch.equal(bad[0][others], grads[0][others])
    assert torch.equal(out[d["ids"] < 0], d["base"][d["ids"] < 0]) and torch.equal(bad[0][d["ids"] < 0], d["dx"][d["ids"] < 0])
    for got, w in zip(bad[1:], grads[1:]):
        assert torch.equal(got[1:], w[1:])
    assert not torch.isfinite(out[d["ids"] == 0]).any(1).all()


def test_scratch_beyond_the_pool():
    """Calls whose scratch does not fit the pool take memory of their own: the same bits, eager, on two streams at once and captured."""
    from rl_engine.kernels.sampling import SamplerBackend

    small, large = SamplerBackend(pool_bytes=1 << 16), SamplerBackend()
    c = {k: v.cuda() for k, v in _inputs(300, 1100, 2000, 40, 3, torch.bfloat16, seed=23).items()}
    args = (c["hidden"], c["a"], c["b"], c["ids"], c["scaling"])
    assert small._lora_workspace_bytes(300, 1100, 2000, 40, 3, 1) > 1 << 20

    def both(backend):
        out, u = backend.lora_linear(c["base"], *args, return_shrunk=True)
        return (out, u, *backend.lora_linear_backward(c["dy"], *args, u, c["dx"]))

    want = both(large)
    side, results = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            results.append(both(small))
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(small)
    for _ in range(3):
        with torch.inference_mode():
            for x in got:
                x.zero_()
        both(small)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("o", [65544, 65541])
def test_many_tokens_in_front_of_a_wide_output(sampler, dtype, o):
    """The size from which the backward takes 1024 outputs per workgroup; the fp64 statement is evaluated on the GPU here."""
    n, h, r, s = 4100, 72, 11, 2
    g = torch.Generator(device="cuda").manual_seed(o)
    rnd = lambda std, *shape: (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)  # noqa: E731
    dy, hidden, a, b, dx_base = rnd(0.1, n, o), rnd(1.0, n, h), rnd(0.1, s, r, h), rnd(0.3, s, o, r), rnd(0.5, n, h)
    ids = torch.randint(-1, s, (n,), generator=g, device="cuda")
    scaling = torch.tensor([0.75, 1.25], device="cuda")
    u = torch.randn(n, r, generator=g, device="cuda")
    got = sampler.lora_linear_backward(dy, hidden, a, b, ids, scaling, u, dx_base)
    with torch.device("cuda"):
        want, bound = lora_ref.backward(dy, hidden, a, b, ids, scaling, u, dx_base)
    for x, w, e, what in zip(got, want, bound, ("dhidden", "dlora_a", "dlora_b")):
        assert ((x.double() - w).abs() - e).max().item() <= 0, what
    again = sampler.lora_linear_backward(dy, hidden, a, b, ids, scaling, u, dx_base)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
