"""verify_draft at the edges of its parameters, against its exact statement in integers (oracle/verify_ref.py)."""
import pytest
import torch

from oracle import verify_ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _equal(sampler, target, ids, u, q, **kw):
    move = lambda t: t.cuda() if isinstance(t, torch.Tensor) else t  # noqa: E731
    got = sampler.verify_draft(target.cuda(), ids.cuda(), u.cuda(), draft_logits=move(q), **{k: move(v) for k, v in kw.items()})
    want = verify_ref.verify(target, ids, u, q, **kw)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [{}, {"top_p": 0.5}, {"top_k": 9}])
@pytest.mark.parametrize("temperature", [1e-37, 2e-38, 1e-3])
def test_temperatures_that_fold_a_row(sampler, dtype, kw, temperature):
    """Rows of negative logits at a temperature so small that every scaled value is -infinity: all of them equal the maximum, those
    of -256 and below and the masked ones too.  A row with a larger entry has that one alone left."""
    vocab, g = 1200, torch.Generator().manual_seed(3)
    pick = torch.tensor([-100.0, -300.0, -float("inf"), -60.0, -90.5])
    row = lambda few: pick[torch.randint(0, len(pick), (vocab,), generator=g)] if few else torch.full((vocab,), -70.0)  # noqa: E731
    for first in (-100.0, -0.25, 0.5):
        for few in (True, False):
            target = torch.stack([torch.stack([row(few) for _ in range(3)]) for _ in range(8)]).to(dtype)
            draft = torch.stack([torch.stack([row(not few) for _ in range(2)]) for _ in range(8)]).to(dtype)
            target[:, :, 5] = first
            ids = torch.randint(0, vocab, (8, 2), generator=g)
            u = torch.rand(8, 3, generator=g)
            _equal(sampler, target, ids, u, draft, temperature=temperature, **kw)
            u[:, :2] *= 3.0 / vocab                           # a looked-up draft is accepted with its probability
            _equal(sampler, target, ids, u, None, temperature=temperature, **kw)


@pytest.mark.parametrize("top_k", [1 << 31, (1 << 32) + 5, (1 << 40) + 1])
def test_top_k_beyond_32_bits_filters_nothing(sampler, top_k):
    g = torch.Generator().manual_seed(4)
    target = torch.randn(6, 3, 500, generator=g).bfloat16()
    draft = torch.randn(6, 2, 500, generator=g).bfloat16()
    ids, u = torch.randint(0, 500, (6, 2), generator=g), torch.rand(6, 3, generator=g)
    plain = sampler.verify_draft(target.cuda(), ids.cuda(), u.cuda(), draft_logits=draft.cuda())
    sampled = sampler.sample(target[:, 0].cuda(), uniforms=u[:, 0].cuda())
    for k in (top_k, torch.full((6,), top_k, dtype=torch.int64, device="cuda")):
        got = sampler.verify_draft(target.cuda(), ids.cuda(), u.cuda(), draft_logits=draft.cuda(), top_k=k)
        assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
        assert torch.equal(sampler.sample(target[:, 0].cuda(), top_k=k, uniforms=u[:, 0].cuda()), sampled)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [{}, {"top_k": 50, "top_p": 0.9}, {"top_p": 0.9}])
def test_uniforms_of_zero(sampler, dtype, kw):
    """u = 0 takes the first entry with mass, by way of the 128-bit draw."""
    g = torch.Generator().manual_seed(6)
    target = (torch.randn(5, 3, 4100, generator=g) * 2).to(dtype)
    draft = (target[:, :2].float() + 0.5 * torch.randn(5, 2, 4100, generator=g)).to(dtype)
    ids = torch.randint(0, 4100, (5, 2), generator=g)
    for q in (draft, None):
        _equal(sampler, target, ids, torch.zeros(5, 3), q, **kw)


def test_log_probability_whatever_the_order_of_the_entries(sampler):
    """Rows with some thousand entries next to zero, which the kernel collects in no fixed order: the same bits for every call and
    for every order of the row's entries."""
    g = torch.Generator().manual_seed(8)
    vocab = 20000
    row = torch.randn(24, vocab, generator=g) * 2
    small = torch.rand(24, vocab, generator=g)
    row = torch.where(small < 0.04, row * 1e-4, torch.where(small < 0.05, torch.zeros(()), row)).bfloat16()
    token = torch.randint(0, vocab, (24, 1), generator=g)
    want = None
    for turn in range(6):
        order = torch.stack([torch.randperm(vocab, generator=g) if turn > 1 else torch.arange(vocab) for _ in range(24)])
        target = row.gather(1, order).unsqueeze(1).expand(24, 2, vocab).contiguous()
        draft = (order == token).nonzero()[:, 1:]
        ids, accepted, lp = sampler.verify_draft(target.cuda(), draft.cuda(), torch.zeros(24, 2).cuda(), return_policy_logprob=True)
        assert (accepted == 1).all() and torch.equal(ids[:, :1].cpu(), draft)
        want = lp[:, 0] if want is None else want
        assert torch.equal(lp[:, 0], want)
    rows = row.double()
    exact = rows.gather(1, token).squeeze(1) - torch.logsumexp(rows, 1)
    assert (want.cpu().double() - exact).abs().max().item() <= 2e-5


@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probabilities_of_rows_far_from_zero(sampler, dtype):
    """Rows whose maximum is some hundreds or thousands, of either sign: to 1e-5 what compute_logp returns, so that a ratio of the two is
    one.  (Both multiply by log2(e) as fp32 and by ln(2) at the end, whose product is off from 1 by 1.3e-8 < 2^-26: against fp64 they are
    off by that much of the row's maximum, beside the tolerance of rows near zero.)"""
    g = torch.Generator().manual_seed(12)
    for top in (300.0, 2000.0, 20000.0, -300.0, -2000.0, -20000.0):
        for vocab in (1, 2, 700, 5000):
            step = 2.0 ** (torch.tensor(abs(top)).log2().floor() - (7 if dtype == torch.bfloat16 else 10))  # of the type, there
            target = (top - step * torch.randint(0, 6, (5, 2, vocab), generator=g)).to(dtype)
            ids = target[:, :1].float().argmax(-1)
            got = sampler.verify_draft(target.cuda(), ids.cuda(), torch.zeros(5, 2).cuda(), return_policy_logprob=True)
            assert torch.equal(got[0][:, :1].cpu(), ids)
            rows = target.double()
            want = rows.gather(2, got[0].cpu().unsqueeze(2)).squeeze(2) - torch.logsumexp(rows, 2)
            assert (got[2].cpu().double() - want).abs().max().item() <= 2e-5 + 2.0 ** -26 * abs(top)
            assert (got[2] - sampler.compute_logp(target.cuda(), got[0])).abs().max().item() <= 1e-5
