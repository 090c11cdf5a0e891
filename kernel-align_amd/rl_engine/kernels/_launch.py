"""What every operator does around a launch: the device check, the device guard, the stream lookup and per-row parameters."""
from __future__ import annotations

import torch


def _require_gpu(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on the GPU: rl_engine has no CPU path (got {t.device})")


class _NoGuard:
    """Stands in for torch.cuda.device(...) when the tensor's device is the current one already."""

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


def _on_device(device):
    """A context manager that makes `device` current for the launch.  Entering torch.cuda.device() and asking
    torch.cuda.current_stream() cost more host time than a small kernel runs, so the common case (the tensor lives
    on the current device) takes neither."""
    index = device.index
    if index is None or index == torch._C._cuda_getDevice():
        return _NO_GUARD
    return torch.cuda.device(index)


def _raw_stream() -> int:
    """Handle of the current HIP stream of the current device (what torch.cuda.current_stream().cuda_stream returns)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def to_rows(values: torch.Tensor, device, dtype) -> torch.Tensor:
    """Per-row parameters in the type the kernels read.  Integers beyond 32 bits become the largest that fit, instead of what their
    low bits say (a top_k beyond the vocabulary filters nothing, however large)."""
    if dtype == torch.int32 and values.dtype in (torch.int64, torch.uint32, torch.uint64):
        limits = torch.iinfo(torch.int32)
        values = values.to(torch.int64).clamp(limits.min, limits.max)
    return values.to(device=device, dtype=dtype).contiguous()
