"""The exact statement of draft verification against closed forms, and against the sampling oracle where the two meet."""
import math
from collections import Counter
from fractions import Fraction

import pytest
import torch

from oracle import exact, verify_ref


def _rows(shape, seed, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * 2.0).to(dtype)


@pytest.mark.parametrize("kw", [{}, {"top_k": 7}, {"top_p": 0.7}, {"top_k": 20, "top_p": 0.8, "temperature": 0.7}])
def test_no_drafts_is_the_sampling_operator(kw):
    target = _rows((6, 1, 97), 3)
    u = torch.rand(6, 1, generator=torch.Generator().manual_seed(4))
    ids, accepted, _ = verify_ref.verify(target, torch.zeros(6, 0, dtype=torch.int64), u, **kw)
    want = exact.sample(target[:, 0], kw.get("temperature", 1.0), kw.get("top_k"), kw.get("top_p"), u[:, 0])
    assert torch.equal(ids[:, 0], want) and accepted.tolist() == [0] * 6


@pytest.mark.parametrize("kw", [{}, {"top_k": 5}, {"top_p": 0.6}])
def test_masses_agree_with_the_sampling_oracle(kw):
    rows = _rows((8, 211), 5)
    _, info = exact.sample(rows, 1.0, kw.get("top_k"), kw.get("top_p"), torch.zeros(8), return_info=True)
    for r in range(8):
        w = verify_ref.row_masses(rows[r], 1.0, **kw)
        assert sum(w) == info[r]["z_kept"] and sum(1 for m in w if m) <= info[r]["n_kept"]


def test_same_rows_accept_everything():
    target = _rows((5, 4, 33), 7)
    draft_ids = torch.stack([exact.sample(target[:, j], 1.0, None, 0.8, torch.rand(5, generator=torch.Generator().manual_seed(j)))
                             for j in range(3)], 1)
    ids, accepted, _ = verify_ref.verify(target, draft_ids, torch.full((5, 4), 1.0), target[:, :3], top_p=0.8)
    assert accepted.tolist() == [3] * 5 and torch.equal(ids[:, :3], draft_ids)


@pytest.mark.parametrize("lookup", [False, True])
def test_emitted_token_is_distributed_as_the_target(lookup):
    """One position, four entries: over all drafts and a grid of uniforms the emitted token's frequencies are P."""
    target = torch.tensor([[[1.0, 0.25, -0.5, 0.0], [0.0, 0.0, 0.0, 0.0]]]).bfloat16()
    draft = torch.tensor([[[0.0, 1.0, 0.5, -1.0]]]).bfloat16()
    wp, wq = verify_ref.row_masses(target[0, 0]), verify_ref.row_masses(draft[0, 0])
    grid = 64
    freq = [Fraction(0)] * 4
    for d in range(4):
        p_d, q_d = Fraction(wp[d], sum(wp)), Fraction(wq[d], sum(wq))
        weight = Fraction(1) if lookup else q_d
        if lookup and d != 2:
            continue
        hits = Counter()
        for a in range(grid):
            for r in range(grid):
                u = torch.tensor([[(a + 0.5) / grid, (r + 0.5) / grid]])
                ids, _, _ = verify_ref.verify(target, torch.tensor([[d]]), u, None if lookup else draft)
                hits[int(ids[0, 0])] += 1
        for i, c in hits.items():
            freq[i] += weight * Fraction(c, grid * grid)
    for i in range(4):
        # every decision boundary falls inside one cell of a grid of 64 x 64: at most 4 boundaries of 1/64 each
        assert abs(float(freq[i] - Fraction(wp[i], sum(wp)))) <= 4.0 / grid


def test_conventions():
    target = _rows((1, 3, 16), 9)
    u0 = torch.zeros(1, 3)
    # an id outside the vocabulary is never accepted, whatever the uniform
    for bad in (-1, 16, 1 << 40):
        ids, accepted, _ = verify_ref.verify(target, torch.tensor([[bad, 0]]), u0)
        assert accepted.item() == 0 and ids[0, 0] >= 0 and ids[0, 1:].tolist() == [-1, -1]
    # a draft that the target filters out is rejected at u = 0, one it keeps is accepted there
    best, worst = int(target[0, 0].float().argmax()), int(target[0, 0].float().argmin())
    assert verify_ref.verify(target, torch.tensor([[worst, 0]]), u0, top_k=3)[1].item() == 0
    assert verify_ref.verify(target, torch.tensor([[best, worst]]), u0, top_k=3)[1].item() == 1
    # a draft that its own row filters out, with the same row as target: no residual, drawn from the target
    same = verify_ref.verify(target, torch.tensor([[worst, 0]]), u0, target[:, :2], top_k=1)
    assert same[1].item() == 0 and same[0][0].tolist() == [best, -1, -1]
    # lengths are clamped
    assert verify_ref.verify(target, torch.tensor([[best, best]]), u0, draft_lens=torch.tensor([-4]))[1].item() == 0
    full = verify_ref.verify(target, torch.tensor([[best, best]]), u0, draft_lens=torch.tensor([99]))
    assert full[1].item() == 2 and (full[0] >= 0).all()
    # the drafter's own mass is respected: P(d) / Q(d) = 1/2 accepts below one half and not above
    t = torch.tensor([[[0.0, 0.0], [0.0, 0.0]]])
    q = torch.tensor([[[0.0, -1000.0]]])
    assert verify_ref.verify(t, torch.tensor([[0]]), torch.tensor([[0.49, 0.3]]), q)[1].item() == 1
    ids, accepted, lp = verify_ref.verify(t, torch.tensor([[0]]), torch.tensor([[0.5, 0.3]]), q)
    assert accepted.item() == 0 and ids[0].tolist() == [1, -1] and lp[0, 0].item() == pytest.approx(-math.log(2.0))
