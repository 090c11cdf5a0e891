"""Refusals of verify_draft, decided on the host (meta tensors stand in for GPU tensors: nothing is launched)."""
import pytest
import torch

from rl_engine.kernels.sampling import SamplerBackend


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it lives on the GPU, so that the checks behind the device check can be reached without one."""
    is_cuda = True


def _fake(t):
    return t.as_subclass(_OnGpu)


def _call(target=None, ids=None, u=None, **kw):
    target = _fake(torch.zeros(2, 4, 16, dtype=torch.bfloat16)) if target is None else target
    ids = torch.zeros(2, 3, dtype=torch.int64) if ids is None else ids
    u = torch.zeros(2, 4) if u is None else u
    return SamplerBackend().verify_draft(target, ids, u, **kw)


@pytest.mark.parametrize("bad, error", [
    (dict(target=torch.zeros(2, 4, 16)), RuntimeError),
    (dict(target=_fake(torch.zeros(4, 16))), ValueError),
    (dict(target=_fake(torch.zeros(2, 0, 16))), ValueError),
    (dict(target=_fake(torch.zeros(2, 4, 0))), ValueError),
    (dict(target=_fake(torch.zeros(2, 4, 16, dtype=torch.float64))), TypeError),
    (dict(target=_fake(torch.zeros(2, 66, 16)), ids=torch.zeros(2, 65, dtype=torch.int64), u=torch.zeros(2, 66)), ValueError),
    (dict(ids=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(ids=torch.zeros(2, 3)), TypeError),
    (dict(ids=torch.zeros(2, 3, dtype=torch.bool)), TypeError),
    (dict(u=torch.zeros(2, 3)), ValueError),
    (dict(draft_lens=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(draft_lens=torch.zeros(2)), TypeError),
    (dict(draft_logits=torch.zeros(2, 3, 16, dtype=torch.bfloat16)), RuntimeError),
    (dict(draft_logits=_fake(torch.zeros(2, 4, 16, dtype=torch.bfloat16))), ValueError),
    (dict(draft_logits=_fake(torch.zeros(2, 3, 16))), TypeError),
    (dict(temperature=0.0), ValueError), (dict(temperature=float("nan")), ValueError), (dict(top_k=0), ValueError),
    (dict(top_p=0.0), ValueError), (dict(top_p=1.01), ValueError), (dict(top_p=torch.ones(3)), ValueError),
])
def test_refusals(bad, error):
    with pytest.raises(error):
        _call(**bad)
