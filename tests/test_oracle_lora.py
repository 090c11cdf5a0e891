"""The fp64 statement of the adapters against autograd, and its gradients against differences."""
import torch

from oracle import lora_ref


def _case(seed=0, n=7, h=5, o=6, r=3, s=3):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64)  # noqa: E731
    return rnd(n, o), rnd(n, h), rnd(s, r, h), rnd(s, o, r), torch.randint(-1, s, (n,), generator=g), torch.rand(s, generator=g) + 0.5


def _token_by_token(base, x, a, b, ids, scale):
    out = []
    for i in range(x.shape[0]):
        y = base[i]
        if ids[i] >= 0:
            k = int(ids[i])
            y = y + float(scale[k]) * (b[k] @ (a[k] @ x[i]))
        out.append(y)
    return torch.stack(out)


def test_forward_and_gradients_against_autograd():
    base, x, a, b, ids, scale = _case()
    y, u, _, _ = lora_ref.forward(base, x, a, b, ids, scale)
    xs, as_, bs = (t.clone().requires_grad_() for t in (x, a, b))
    want = _token_by_token(base, xs, as_, bs, ids, scale)
    assert torch.allclose(y, want, rtol=1e-13, atol=1e-13)
    dy = torch.randn(want.shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
    want.backward(dy)
    (dx, da, db), _ = lora_ref.backward(dy, x, a, b, ids, scale, u, None)
    for got, leaf in ((dx, xs), (da, as_), (db, bs)):
        assert torch.allclose(got, leaf.grad, rtol=1e-12, atol=1e-13)


def test_gradients_against_differences():
    base, x, a, b, ids, scale = _case(seed=3, n=4, s=2)
    dy = torch.randn(base.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    u = lora_ref.forward(base, x, a, b, ids, scale)[1]
    (dx, da, db), _ = lora_ref.backward(dy, x, a, b, ids, scale, u, None)
    step = 1e-6
    for leaf, grad in ((x, dx), (a, da), (b, db)):
        flat = leaf.view(-1)
        for i in range(0, flat.numel(), 5):
            keep = flat[i].item()
            flat[i] = keep + step
            up = (lora_ref.forward(base, x, a, b, ids, scale)[0] * dy).sum()
            flat[i] = keep - step
            down = (lora_ref.forward(base, x, a, b, ids, scale)[0] * dy).sum()
            flat[i] = keep
            # central difference: truncation is zero (bilinear in each leaf), cancellation 2^-52 of a sum of order 100 over 2e-6
            assert abs((up - down).item() / (2 * step) - grad.view(-1)[i].item()) <= 1e-7


def test_tokens_without_an_adapter():
    base, x, a, b, _, scale = _case(seed=5)
    ids = torch.full((7,), -1)
    y, u, _, _ = lora_ref.forward(base, x, a, b, ids, scale)
    assert torch.equal(y, base) and not u.any()
    (dx, da, db), _ = lora_ref.backward(base, x, a, b, ids, scale, u, x)
    assert torch.equal(dx, x) and not da.any() and not db.any()
