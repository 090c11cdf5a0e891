"""The names, the rollout loop and the training nodes around verification and adapters: what is decided on the host."""
import pytest
import torch

from rl_engine.executors.rollout import RolloutExecutor
from rl_engine.kernels import autograd
from rl_engine.kernels.registry import OpBackend, kernel_registry
from rl_engine.kernels.sampling import SamplerBackend


def test_names_resolve_to_the_operators():
    for name in ("verify_draft", "draft_verification", "verification"):
        assert kernel_registry.dispatch(name) == "HIP_VERIFY_DRAFT"
    for name in ("lora", "lora_linear", "lora_lm_head", "adapter"):
        assert kernel_registry.dispatch(name) == "HIP_LORA_LINEAR"
    assert kernel_registry.dispatch("linear") == "HIP_FUSED_LMHEAD_LOGPROB"
    assert kernel_registry.dispatch("speculative_sampling") == "HIP_SAMPLING"
    assert kernel_registry.get_op_path(OpBackend.HIP_VERIFY_DRAFT).endswith("SamplerBackend.verify_draft")
    assert kernel_registry.resolve("verify_draft").__name__ == "verify_draft"
    assert kernel_registry.resolve("lora_linear").__name__ == "lora_linear"


def test_speculative_generation_checks_its_arguments_and_never_falls_back_to_the_cpu():
    executor = RolloutExecutor({"top_k": 4})
    ids = torch.zeros(2, 3, dtype=torch.int64)
    drafts = (torch.zeros(2, 2, dtype=torch.int64), None)
    with pytest.raises(ValueError, match="prompt_ids"):
        executor.generate_speculative(None, None, torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match="uniforms"):
        executor.generate_speculative(None, None, ids, 2, uniforms=torch.zeros(3, 2, 4))
    with pytest.raises(RuntimeError):
        executor.generate_speculative(lambda *a: torch.zeros(2, 3, 16), lambda *a: drafts, ids, 2)
    out, lp, passes = executor.generate_speculative(None, None, ids, 0)
    assert torch.equal(out, ids) and lp.shape == (2, 0) and passes == 0


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it lives on the GPU, so that the checks behind the device check can be reached without one."""
    is_cuda = True


def _fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnGpu)


def _logp_args(**change):
    args = dict(hidden=_fake(4, 5), weight=_fake(6, 5), lora_a=_fake(2, 3, 5), lora_b=_fake(2, 6, 3),
                token_ids=torch.zeros(4, dtype=torch.int64), adapter_ids=torch.zeros(4, dtype=torch.int64))
    args.update(change)
    return args


@pytest.mark.parametrize("change, error", [
    (dict(hidden=torch.zeros(4, 5, dtype=torch.bfloat16)), RuntimeError),
    (dict(weight=_fake(7, 5)), ValueError),
    (dict(weight=_fake(6, 4)), ValueError),
    (dict(weight=_fake(6, 5, dtype=torch.float16)), TypeError),
    (dict(weight=torch.zeros(6, 5, dtype=torch.bfloat16)), RuntimeError),
    (dict(weight=torch.zeros(6, 5, dtype=torch.bfloat16).requires_grad_(True).as_subclass(_OnGpu)), ValueError),
    (dict(token_ids=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(adapter_ids=torch.zeros(4, 1, dtype=torch.int64)), ValueError),
    (dict(chunk_tokens=0), ValueError),
    (dict(scaling=torch.ones(2, requires_grad=True)), ValueError),
    (dict(scaling=torch.ones(3)), ValueError),
])
def test_refusals_of_the_training_nodes(change, error):
    with pytest.raises(error):
        autograd.lora_linear_logp(SamplerBackend(), **_logp_args(**change))


def test_scaling_has_no_gradient():
    with pytest.raises(ValueError, match="scaling"):
        autograd.lora_linear(None, None, None, None, None, None, torch.ones(2, requires_grad=True))
