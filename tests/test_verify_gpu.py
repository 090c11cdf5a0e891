"""verify_draft on the GPU against its exact statement in integers (oracle/verify_ref.py).  Ids and counts are equal; the
policy log-probabilities are held to 2e-5 against fp64, as those of compute_logp are (fp32 sums of a row, one rounding of a value
below 2^6: 2^-19 at most of it)."""
import pytest
import torch

from oracle import verify_ref

pytestmark = pytest.mark.gpu

LOGP_TOL = 2e-5
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(batch, k, vocab, dtype, seed, draft=True, ragged=False, sigma=2.0, noise=0.5):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(batch, k + 1, vocab, generator=g) * sigma
    target = base.to(dtype)
    q = (base[:, :k] + noise * torch.randn(batch, k, vocab, generator=g)).to(dtype) if draft else None
    # drafts from the drafter's softmax (or the target's, without one), some of them any token
    src = (q if draft else target[:, :k]).float()
    ids = torch.multinomial(torch.softmax(src.reshape(batch * k, vocab), -1), 1, generator=g).view(batch, k) if k else \
        torch.zeros(batch, 0, dtype=torch.int64)
    wild = torch.rand(batch, k, generator=g) < 0.1
    ids = torch.where(wild, torch.randint(0, vocab, (batch, k), generator=g), ids)
    u = torch.rand(batch, k + 1, generator=g)
    lens = torch.randint(-1, k + 2, (batch,), generator=g) if ragged else None
    return target, ids, u, q, lens


def _gpu(t):
    return None if t is None else t.cuda()


def _check(sampler, target, ids, u, q, lens, **kw):
    gkw = {n: _gpu(v) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    got = sampler.verify_draft(_gpu(target), _gpu(ids), _gpu(u), draft_logits=_gpu(q), draft_lens=_gpu(lens),
                               return_policy_logprob=True, **gkw)
    want = verify_ref.verify(target, ids, u, q, lens, **kw)
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0])
    lp = got[2].cpu().double()
    both = torch.isfinite(want[2])
    assert torch.equal(torch.isfinite(lp), both)
    assert (lp - want[2])[both].abs().max().item() <= LOGP_TOL if both.any() else True
    return got


FILTERS = [{}, {"temperature": 0.7}, {"top_k": 5}, {"top_k": 50, "top_p": 0.9, "temperature": 0.7}, {"top_p": 0.6},
           {"top_p": 0.95, "temperature": 1.3}, {"top_k": 700, "top_p": 0.8}]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", FILTERS)
@pytest.mark.parametrize("vocab", [1000, 1003])
def test_matches_the_exact_statement(sampler, dtype, kw, vocab):
    for draft in (True, False):
        _check(sampler, *_inputs(6, 3, vocab, dtype, seed=vocab + 7 * draft, draft=draft, ragged=True), **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 64, 65, 513, 8191, 8192, 8193, 32000])
def test_vocabulary_sizes(sampler, dtype, vocab):
    for kw in ({}, {"top_k": 3, "top_p": 0.9}, {"top_p": 0.5}):
        _check(sampler, *_inputs(3, 2, vocab, dtype, seed=vocab), **kw)


@pytest.mark.parametrize("k", [0, 1, 5, 63, 64])
def test_numbers_of_drafts(sampler, k):
    t, ids, u, q, lens = _inputs(3, k, 130, torch.bfloat16, seed=k, ragged=k > 1, noise=0.05)
    _check(sampler, t, ids, u * 0.5, q if k else None, lens, top_p=0.9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_full_size_rows(sampler, dtype):
    """128,256 entries, drafts accepted and rejected at several positions, every filter that the repository benchmarks."""
    for seed, kw in enumerate(({}, {"temperature": 0.7, "top_k": 50, "top_p": 0.9}, {"temperature": 0.7, "top_p": 0.9})):
        got = _check(sampler, *_inputs(2, 2, 128256, dtype, seed=seed, sigma=3.0, noise=0.3), **kw)
        assert got[0].shape == (2, 3)


def test_no_draft_is_sample(sampler):
    g = torch.Generator().manual_seed(1)
    logits = (torch.randn(40, 1, 32000, generator=g) * 3).bfloat16().cuda()
    u = torch.rand(40, 1, generator=g).cuda()
    none = torch.zeros(40, 0, dtype=torch.int64, device="cuda")
    for kw in FILTERS:
        ids, accepted, lp = sampler.verify_draft(logits, none, u, return_policy_logprob=True, **kw)
        want, policy = sampler.sample(logits[:, 0], uniforms=u[:, 0], return_policy_logprob=True, **kw)
        assert torch.equal(ids[:, 0], want) and not accepted.any()
        assert (lp[:, 0] - policy).abs().max().item() <= 1e-5


def _special_rows(dtype, vocab=640):
    inf = float("inf")
    g = torch.Generator().manual_seed(11)
    normal = torch.randn(vocab, generator=g) * 2
    rows = {"equal": torch.zeros(vocab), "all -inf": torch.full((vocab,), -inf),
            "one left": torch.full((vocab,), -inf).index_fill(0, torch.tensor([17]), 3.0),
            "masked": torch.where(torch.rand(vocab, generator=g) < 0.7, torch.tensor(-inf), normal),
            "lowest": torch.where(torch.rand(vocab, generator=g) < 0.7, torch.tensor(torch.finfo(dtype).min), normal),
            "+inf": normal.clone().index_fill(0, torch.tensor([3, 400]), inf),
            "nan": normal.clone().index_fill(0, torch.tensor([5, 6, 630]), float("nan")),
            "few values": torch.round(normal), "tiny": normal * 1e-3, "large": normal * 300.0,
            "huge": torch.full((vocab,), 200.0) + torch.round(normal) * 64, "negative": -torch.round(normal.abs() * 4) - 300.0,
            "signed zeros": torch.where(torch.rand(vocab, generator=g) < 0.5, torch.tensor(0.0), torch.tensor(-0.0))}
    return {k: v.to(dtype) for k, v in rows.items()}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [{}, {"temperature": 0.6}, {"temperature": 40.0, "top_k": 9}, {"top_k": 20, "top_p": 0.7},
                                {"top_p": 0.5}, {"top_p": 0.999}])
def test_special_rows(sampler, dtype, kw):
    """Masked rows, rows with nothing left, ties, infinities, NaN, values far from zero: each as target and as draft."""
    rows = _special_rows(dtype)
    names = sorted(rows)
    g = torch.Generator().manual_seed(5)
    target = torch.stack([torch.stack([rows[n], rows["masked"]]) for n in names for _ in range(4)])
    draft = torch.stack([rows[names[(i + s) % len(names)]].unsqueeze(0) for i in range(len(names)) for s in range(4)])
    batch, vocab = target.shape[0], target.shape[2]
    ids = torch.randint(0, vocab, (batch, 1), generator=g)
    best = torch.nan_to_num(target[:, 0].float(), nan=-1e38).argmax(-1, keepdim=True)
    ids = torch.where(torch.rand(batch, 1, generator=g) < 0.5, best, ids)
    u = torch.rand(batch, 2, generator=g)
    # (the log-probability of a row with +inf or NaN is not a number; ids are what counts here)
    gkw = dict(kw)
    for q in (draft, None):
        got = sampler.verify_draft(target.cuda(), ids.cuda(), u.cuda(), draft_logits=_gpu(q), **gkw)
        want = verify_ref.verify(target, ids, u, q, **kw)
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])


@pytest.mark.parametrize("kw", [{}, {"temperature": 0.6}, {"top_p": 0.5}, {"top_p": 0.97, "temperature": 1.3}, {"top_k": 2000}])
def test_special_rows_of_a_large_vocabulary(sampler, kw):
    """bf16 rows long enough for the tables of the last pass, with values outside their bins: tiny ones of both signs, zeros,
    masked entries, values far from zero - and the same as drafts."""
    rows = _special_rows(torch.bfloat16, vocab=40004)
    del rows["one left"]
    g = torch.Generator().manual_seed(15)
    rows["tiny and not"] = torch.where(torch.rand(40004, generator=g) < 0.02, torch.randn(40004, generator=g) * 3e-4,
                                       torch.randn(40004, generator=g)).bfloat16()
    names = sorted(rows)
    target = torch.stack([torch.stack([rows[n], rows["masked"]]) for n in names for _ in range(2)])
    draft = torch.stack([rows[names[(i + s) % len(names)]].unsqueeze(0) for i in range(len(names)) for s in (0, 5)])
    batch, vocab = target.shape[0], target.shape[2]
    ids = torch.randint(0, vocab, (batch, 1), generator=g)
    u = torch.rand(batch, 2, generator=g)
    for q in (draft, None):
        got = sampler.verify_draft(target.cuda(), ids.cuda(), u.cuda(), draft_logits=_gpu(q), **kw)
        want = verify_ref.verify(target, ids, u, q, **kw)
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_draws_on_a_border(sampler, dtype):
    """Rows of equal masses whose uniform falls exactly on the border between two entries: decided in integers."""
    t = torch.zeros(8, 2, 4096, dtype=dtype)
    q = t[:, :1].clone()
    u = torch.zeros(8, 2)
    u[:, 1] = torch.arange(8) / 8.0
    ids = torch.arange(8).unsqueeze(1)
    got = _check(sampler, t, ids, u, q, None)
    assert got[1].tolist() == [1] * 8 and got[0][:, 1].tolist() == [512 * i for i in range(8)]
    _check(sampler, t[:, :1], ids[:, :0], u[:, 1:], None, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_at_the_cut(sampler, dtype):
    """Rows of a handful of values: top-p cuts inside a group of equal logits, and the drafts sit in that group on both sides
    of the cut, in the target and in the drafter's row."""
    g = torch.Generator().manual_seed(21)
    batch, k, vocab = 24, 2, 2050
    target = torch.randint(0, 3, (batch, k + 1, vocab), generator=g).to(dtype)
    draft = torch.randint(0, 3, (batch, k, vocab), generator=g).to(dtype)
    ids = torch.randint(0, vocab, (batch, k), generator=g)
    u = torch.rand(batch, k + 1, generator=g) * 0.9
    for kw in ({"top_p": 0.3}, {"top_p": 0.8}, {"top_k": 40, "top_p": 0.5}, {"top_k": 40}):
        _check(sampler, target, ids, u, draft, None, **kw)
        _check(sampler, target, ids, u, None, None, **kw)


def test_uniforms_at_their_ends_and_ids_outside(sampler):
    t, ids, u, q, _ = _inputs(12, 3, 300, torch.bfloat16, seed=2)
    ids[0, 0], ids[1, 1], ids[2, 2], ids[3, 0] = -1, 300, 1 << 40, -(1 << 40)
    for value in (0.0, 1.0, -3.0, float("nan"), 1e-45, 1.0 - 2.0 ** -24):
        _check(sampler, t, ids, torch.full_like(u, value), q, None, top_p=0.9)
        _check(sampler, t, ids, torch.full_like(u, value), None, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_residual_is_drawn_from_the_target(sampler, dtype):
    """The same row as target and as draft, with a draft that the filters drop: P - Q is zero everywhere."""
    g = torch.Generator().manual_seed(13)
    t = (torch.randn(6, 2, 20003, generator=g) * 2).to(dtype)
    ids = t[:, 0].float().argmin(-1, keepdim=True)
    ids[5] = -1
    u = torch.rand(6, 2, generator=g)
    for kw in ({"top_k": 40}, {"top_p": 0.9}, {"top_k": 1}):
        got = _check(sampler, t, ids, u, t[:, :1].clone(), None, **kw)
        want = sampler.sample(t[:, 0].cuda(), uniforms=u[:, 1].cuda(), **kw)
        assert torch.equal(got[0][:, 0], want) and not got[1].any()


def test_per_request_parameters(sampler):
    t, ids, u, q, lens = _inputs(7, 2, 515, torch.bfloat16, seed=8, ragged=True)
    temp = torch.tensor([1.0, 0.7, 0.0, 2.0, float("nan"), 0.3, 1.1])
    top_k = torch.tensor([0, 5, 50, -2, 1, 600, 20])
    top_p = torch.tensor([1.0, 0.9, 0.0, 0.5, 1.5, 0.2, 0.95])
    _check(sampler, t, ids, u, q, lens, temperature=temp, top_k=top_k, top_p=top_p)
    _check(sampler, t, ids, u, None, lens, temperature=0.8, top_k=top_k)


def test_layouts(sampler):
    """Views with gaps, odd offsets and transposed positions give what their copies give."""
    g = torch.Generator().manual_seed(3)
    big = (torch.randn(4, 5, 1030, generator=g) * 2).bfloat16().cuda()
    ids = torch.randint(0, 1000, (4, 2), generator=g).cuda()
    u = torch.rand(4, 3, generator=g).cuda() * 0.3
    for target, draft in ((big[:, :3, :1000], big[:, 2:4, 3:1003]), (big[:, 1:4, 1:1001], big[:, ::2][:, :2, 8:1008]),
                          (big.transpose(0, 1)[:3, :3, :1000], big.transpose(0, 1)[1:4, 1:3, 5:1005]),
                          (big[..., ::1].transpose(1, 2)[:, :3, :5], big.transpose(1, 2)[:, 3:5, :5])):
        b = target.shape[0]
        tok = ids[:b] % target.shape[2]
        got = sampler.verify_draft(target, tok, u[:b], draft_logits=draft, top_p=0.9, return_policy_logprob=True)
        want = sampler.verify_draft(target.contiguous(), tok, u[:b], draft_logits=draft.contiguous(), top_p=0.9,
                                    return_policy_logprob=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        # the summation order of a log-sum-exp depends on the alignment of its row
        assert (got[2] - want[2]).abs().max().item() <= 1e-5


def test_rows_behind_the_drafts_are_not_read(sampler):
    t, ids, u, q, _ = _inputs(3, 3, 256, torch.bfloat16, seed=4)
    lens = torch.tensor([0, 1, 2])
    want = sampler.verify_draft(t.cuda(), ids.cuda(), u.cuda(), draft_logits=q.cuda(), draft_lens=lens.cuda())
    for b in range(3):
        t[b, lens[b] + 1:] = float("nan")
        q[b, lens[b]:] = float("nan")
        ids[b, lens[b]:] = 1 << 50
    got = sampler.verify_draft(t.cuda(), ids.cuda(), u.cuda(), draft_logits=q.cuda(), draft_lens=lens.cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_batch_and_launch_do_not_matter(sampler):
    t, ids, u, q, _ = _inputs(300, 1, 2000, torch.bfloat16, seed=6)
    args = (t.cuda(), ids.cuda(), u.cuda(), q.cuda())
    whole = sampler.verify_draft(*args[:3], draft_logits=args[3], top_p=0.9, return_policy_logprob=True)
    for b in (0, 17, 299):
        part = sampler.verify_draft(*(a[b:b + 1] for a in args[:3]), draft_logits=args[3][b:b + 1], top_p=0.9,
                                    return_policy_logprob=True)
        assert all(torch.equal(x[b:b + 1], y) for x, y in zip(whole, part))


def test_graph_replay_and_two_streams(sampler):
    """Captured calls own their workspace: replays with eager calls on another stream in between give the eager results."""
    sets = [[x.cuda() for x in _inputs(9, 3, 4096, torch.bfloat16, seed=s)[:4]] for s in range(3)]
    kw = dict(top_k=30, top_p=0.8, temperature=0.7, return_policy_logprob=True)
    want = [sampler.verify_draft(s[0], s[1], s[2], draft_logits=s[3], **kw) for s in sets]
    buf = [x.clone() for x in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sampler.verify_draft(buf[0], buf[1], buf[2], draft_logits=buf[3], **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sampler.verify_draft(buf[0], buf[1], buf[2], draft_logits=buf[3], **kw)
    for i in (0, 1, 2, 1, 0):
        for dst, src in zip(buf, sets[i]):
            dst.copy_(src)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = sampler.verify_draft(*sets[(i + 1) % 3][:3], draft_logits=sets[(i + 1) % 3][3], **kw)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        assert all(torch.equal(a, b) for a, b in zip(other, want[(i + 1) % 3]))


def test_generator_and_empty_batch(sampler):
    t, ids, _, q, _ = _inputs(4, 2, 128, torch.float16, seed=9)
    g = torch.Generator(device="cuda").manual_seed(7)
    a = sampler.verify_draft(t.cuda(), ids.cuda(), draft_logits=q.cuda(), generator=g)
    u = torch.rand(4, 3, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    b = sampler.verify_draft(t.cuda(), ids.to(torch.int32).cuda(), u, draft_logits=q.cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    e = sampler.verify_draft(t[:0].cuda(), ids[:0].cuda(), u[:0], return_policy_logprob=True)
    assert e[0].shape == (0, 3) and e[1].shape == (0,) and e[2].shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_worked_on_by_several_workgroups(sampler, dtype):
    """A call of few long rows and the same requests inside a call of many take different routes to the same bits, for requests with
    and without top-k side by side, odd lengths, masked entries, and rows that the bins do not describe."""
    vocab, k = 40003, 3
    target, ids, u, q, lens = _inputs(60, k, vocab, dtype, 31, ragged=True)
    target[1, 0, 7:20000] = -float("inf")
    target[2, 1, :] = torch.finfo(dtype).min
    target[2, 1, 11] = 3.0
    target[3, 0, 5] = float("nan")
    target[4, 1, 9] = 1000.0
    top_k = torch.zeros(60, dtype=torch.int32)
    top_k[::3] = 40
    top_p = torch.linspace(0.3, 1.0, 60)
    kw = dict(top_k=top_k, top_p=top_p, temperature=0.8)
    d = [None if t is None else t.cuda() for t in (target, ids, u, q, lens)]
    few = [slice(0, 6), slice(6, 7), slice(40, 60)]
    many = sampler.verify_draft(d[0], d[1], d[2], draft_logits=d[3], draft_lens=d[4], return_policy_logprob=True, **kw)
    for part in few:
        sub = dict(kw, top_k=top_k[part], top_p=top_p[part])
        got = sampler.verify_draft(d[0][part], d[1][part], d[2][part], draft_logits=d[3][part], draft_lens=d[4][part],
                                   return_policy_logprob=True, **sub)
        assert torch.equal(got[0], many[0][part]) and torch.equal(got[1], many[1][part])
        assert torch.equal(got[2].view(torch.int32), many[2][part].view(torch.int32))
    part = slice(0, 6)
    want = verify_ref.verify(target[part], ids[part], u[part], q[part], lens[part], temperature=0.8, top_k=top_k[part], top_p=top_p[part])
    assert torch.equal(many[0][part].cpu(), want[0]) and torch.equal(many[1][part].cpu(), want[1])
