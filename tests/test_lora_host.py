"""Refusals of the adapter operators, decided on the host: nothing is launched."""
import pytest
import torch

from rl_engine.kernels.sampling import SamplerBackend


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it lives on the GPU, so that the checks behind the device check can be reached without one."""
    is_cuda = True


def _fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnGpu)


def _args(**change):
    args = dict(base=_fake(4, 6), hidden=_fake(4, 5), lora_a=_fake(2, 3, 5), lora_b=_fake(2, 6, 3),
                adapter_ids=torch.zeros(4, dtype=torch.int64))
    args.update(change)
    return args


BAD = [
    (dict(hidden=torch.zeros(4, 5)), RuntimeError),
    (dict(lora_a=torch.zeros(2, 3, 5)), RuntimeError),
    (dict(hidden=_fake(4, 5, dtype=torch.float32), lora_a=_fake(2, 3, 5, dtype=torch.float32),
          lora_b=_fake(2, 6, 3, dtype=torch.float32)), TypeError),
    (dict(lora_b=_fake(2, 6, 3, dtype=torch.float16)), TypeError),
    (dict(hidden=_fake(4, 7)), ValueError),
    (dict(lora_a=_fake(3, 5)), ValueError),
    (dict(lora_b=_fake(3, 6, 3)), ValueError),
    (dict(lora_b=_fake(2, 6, 4)), ValueError),
    (dict(lora_a=_fake(2, 129, 5), lora_b=_fake(2, 6, 129)), ValueError),
    (dict(lora_a=_fake(1024, 3, 5), lora_b=_fake(1024, 6, 3)), ValueError),
    (dict(lora_a=_fake(0, 3, 5), lora_b=_fake(0, 6, 3)), ValueError),
    (dict(adapter_ids=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(adapter_ids=torch.zeros(4)), TypeError),
    (dict(adapter_ids=torch.zeros(4, dtype=torch.bool)), TypeError),
    (dict(scaling=torch.ones(3)), ValueError),
]


@pytest.mark.parametrize("change, error", BAD + [(dict(base=_fake(4, 7)), ValueError), (dict(base=torch.zeros(4, 6)), RuntimeError),
                                                 (dict(base=_fake(4, 6, dtype=torch.float16)), TypeError)])
def test_forward_refusals(change, error):
    with pytest.raises(error):
        SamplerBackend().lora_linear(**_args(**change))


@pytest.mark.parametrize("change, error", BAD + [
    (dict(grad_out=_fake(4, 5)), ValueError), (dict(grad_out=_fake(4, 6, dtype=torch.float16)), TypeError),
    (dict(dhidden_base=_fake(4, 6)), ValueError), (dict(dhidden_base=torch.zeros(4, 5)), RuntimeError),
    (dict(shrunk=_fake(4, 3)), TypeError), (dict(shrunk=_fake(4, 4, dtype=torch.float32)), ValueError)])
def test_backward_refusals(change, error):
    args = _args(**change)
    args.pop("base")
    args.setdefault("grad_out", _fake(4, 6))
    with pytest.raises(error):
        SamplerBackend().lora_linear_backward(**args)
