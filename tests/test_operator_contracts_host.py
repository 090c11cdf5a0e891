"""What the entry points around verification, adapters and the registry promise, as far as the host decides it."""
import pytest
import torch

from rl_engine.kernels import _hip
from rl_engine.kernels._launch import to_rows
from rl_engine.kernels.registry import kernel_registry
from rl_engine.kernels.sampling import SamplerBackend


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it lives on the GPU, so that the checks behind the device check can be reached without one."""
    is_cuda = True


def _fake(*shape, dtype=torch.bfloat16, grad=False):
    return torch.zeros(*shape, dtype=dtype).requires_grad_(grad).as_subclass(_OnGpu)


def test_names_of_other_operators_keep_their_answers():
    """A name is the adapters' where one of its words says so, and none of the operators around them does."""
    for name, want in (("exploration_logp", "HIP_LOGPROB"), ("exploration_linear", "HIP_FUSED_LMHEAD_LOGPROB"),
                       ("adapter_linear_logp", "HIP_FUSED_LMHEAD_LOGPROB"), ("lora_linear_logp", "HIP_FUSED_LMHEAD_LOGPROB"),
                       ("adapter_logp", "HIP_LOGPROB"), ("adapter_sampling", "HIP_SAMPLING"), ("exploration_sampling", "HIP_SAMPLING"),
                       ("exploration", "NOT_ON_HIP_PATH"), ("lora", "HIP_LORA_LINEAR"), ("multi-lora", "HIP_LORA_LINEAR"),
                       ("adapters", "HIP_LORA_LINEAR"), ("lora.linear", "HIP_LORA_LINEAR")):
        assert kernel_registry.dispatch(name) == want, name


def test_in_place_refuses_a_leaf_that_requires_grad():
    args = (_fake(4, 5), _fake(2, 3, 5), _fake(2, 6, 3), torch.zeros(4, dtype=torch.int64))
    leaf = torch.zeros(4, 6, dtype=torch.bfloat16, requires_grad=True)
    leaf.__class__ = _OnGpu
    assert leaf.is_leaf and leaf.requires_grad
    view = torch.zeros(4, 8, dtype=torch.bfloat16, requires_grad=True)[:, :6]
    view.__class__ = _OnGpu
    for base in (leaf, view):
        with pytest.raises(ValueError, match="leaf"):
            SamplerBackend().lora_linear(base, *args, inplace=True)


def test_verify_workspace_query_refuses_what_the_call_refuses():
    ws = _hip.load().ka_verify_workspace_bytes
    assert ws(0, 65535, 1, 100) > 0 and ws(2, 4, 64, 100) > 0
    assert ws(3, 4, 4, 100) == 0 and ws(-1, 4, 4, 100) == 0              # no such type
    assert ws(0, 65536, 1, 100) == 0 and ws(0, 65535, 64, 100) == 0      # more requests, more rows than a call takes


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.uint8, torch.uint16, torch.uint32, torch.uint64, torch.float32,
                                   torch.float16])
def test_row_parameters_of_every_type(dtype):
    """Small values as they are, in any type; those beyond 32 bits as the largest that fit."""
    got = to_rows(torch.tensor([0, 5, 100], dtype=torch.int64).to(dtype), torch.device("cpu"), torch.int32)
    assert got.dtype == torch.int32 and got.tolist() == [0, 5, 100]
    if dtype in (torch.int64, torch.uint32):
        big = torch.tensor([(1 << 31) + 5, 7], dtype=torch.int64).to(dtype)
        assert to_rows(big, torch.device("cpu"), torch.int32).tolist() == [(1 << 31) - 1, 7]
    if dtype == torch.int64:
        wide = torch.tensor([(1 << 32) + 5, -(1 << 40)])
        assert to_rows(wide, torch.device("cpu"), torch.int32).tolist() == [(1 << 31) - 1, -(1 << 31)]
