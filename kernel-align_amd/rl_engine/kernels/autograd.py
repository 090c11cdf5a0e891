"""Differentiable wrappers of the logprob operators for training loops.

The reference's operators run under ``torch.inference_mode()`` (rl_engine/kernels/sampling.py:38,91) and
cannot be part of a graph.  These ``torch.autograd.Function`` s put the same kernels into one:

    logp = logp_from_logits(sampler, logits, token_ids)          # d/dlogits
    logp = linear_logp(sampler, hidden, weight, token_ids)       # d/dhidden, d/dweight; logits never stored
    out = lora_linear(sampler, base, hidden, lora_a, lora_b, adapter_ids)                   # d/dbase, hidden, lora_a, lora_b
    logp = lora_linear_logp(sampler, hidden, weight, lora_a, lora_b, token_ids, adapter_ids)  # weight frozen, logits never stored

Forward and backward both run on the HIP kernels; nothing here computes on the CPU.  A training step may be captured in a
HIP graph, forward and backward together; as with every torch module, no eager graph of the same leaves may be alive then.
"""
from __future__ import annotations

import torch

from rl_engine.kernels._launch import _require_gpu
from rl_engine.kernels.sampling import LMHEAD_BACKWARD_CHUNK_TOKENS, _chunk_rows


class _LogpFromLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, sampler, logits, token_ids):
        logp = sampler._compute_logp(logits, token_ids)
        ctx.sampler = sampler
        ctx.save_for_backward(logits, token_ids, logp)
        return logp

    @staticmethod
    def backward(ctx, grad_logp):
        logits, token_ids, logp = ctx.saved_tensors
        dlogits = ctx.sampler._compute_logp_backward(logits, token_ids, logp, grad_logp.contiguous())
        return None, dlogits, None


class _LinearLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, sampler, hidden, weight, token_ids, chunk_tokens):
        logp = sampler._fused_linear_logp(hidden, weight, token_ids)
        ctx.sampler = sampler
        ctx.chunk_tokens = chunk_tokens
        ctx.save_for_backward(hidden, weight, token_ids)
        return logp

    @staticmethod
    def backward(ctx, grad_logp):
        hidden, weight, token_ids = ctx.saved_tensors
        dhidden, dweight = ctx.sampler._fused_linear_logp_backward(
            hidden, weight, token_ids, grad_logp.contiguous(), ctx.chunk_tokens)
        return None, dhidden, dweight.to(weight.dtype), None, None


def logp_from_logits(sampler, logits: torch.Tensor, token_ids: torch.Tensor) -> torch.Tensor:
    """``compute_logp`` as a node of the autograd graph: fp32 [..], gradient flows to ``logits``."""
    return _LogpFromLogits.apply(sampler, logits, token_ids)


def linear_logp(sampler, hidden: torch.Tensor, weight: torch.Tensor, token_ids: torch.Tensor,
                chunk_tokens: int | None = None) -> torch.Tensor:
    """``fused_linear_logp`` as a node of the autograd graph: gradients flow to ``hidden`` and ``weight``.

    The backward pass rebuilds the logits one chunk of ``chunk_tokens`` rows at a time, so the peak extra
    memory is one chunk of bf16 logits plus the fp32 weight-gradient accumulator.
    """
    return _LinearLogp.apply(sampler, hidden, weight, token_ids, chunk_tokens)


class _LoraLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, sampler, base, hidden, lora_a, lora_b, adapter_ids, scaling):
        out, shrunk = sampler._lora_linear(base, hidden, lora_a, lora_b, adapter_ids, scaling, return_shrunk=True)
        ctx.sampler = sampler
        ctx.scale = None if isinstance(scaling, torch.Tensor) else scaling
        ctx.save_for_backward(hidden, lora_a, lora_b, adapter_ids, shrunk, *([] if ctx.scale is not None else [scaling]))
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        hidden, lora_a, lora_b, adapter_ids, shrunk, *scaling = ctx.saved_tensors
        needs = ctx.needs_input_grad
        dhidden = da = db = None
        if any(needs[2:5]):
            dhidden, da, db = ctx.sampler._lora_linear_backward(
                grad_out, hidden, lora_a, lora_b, adapter_ids, scaling[0] if scaling else ctx.scale, shrunk)
            da, db = da.to(lora_a.dtype), db.to(lora_b.dtype)
        return (None, grad_out if needs[1] else None, dhidden if needs[2] else None, da if needs[3] else None,
                db if needs[4] else None, None, None)


class _LoraLinearLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, sampler, hidden, weight, lora_a, lora_b, token_ids, adapter_ids, scaling, chunk_tokens):
        logp = torch.empty(hidden.shape[:-1], dtype=torch.float32, device=hidden.device)
        rows, tokens, adapters = _lora_rows(hidden, token_ids, adapter_ids)
        for part in _chunks(rows.shape[0], chunk_tokens):
            logits = torch.matmul(rows[part], weight.t())
            sampler._lora_linear(logits, rows[part], lora_a, lora_b, adapters[part], scaling, inplace=True)
            logp.view(-1)[part] = sampler._compute_logp(logits, tokens[part])
            del logits
        ctx.sampler, ctx.chunk_tokens = sampler, chunk_tokens
        ctx.scale = None if isinstance(scaling, torch.Tensor) else scaling
        ctx.save_for_backward(hidden, weight, lora_a, lora_b, token_ids, adapter_ids,
                              *([] if ctx.scale is not None else [scaling]))
        return logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logp):
        hidden, weight, lora_a, lora_b, token_ids, adapter_ids, *scaling = ctx.saved_tensors
        scaling = scaling[0] if scaling else ctx.scale
        sampler = ctx.sampler
        rows, tokens, adapters = _lora_rows(hidden, token_ids, adapter_ids)
        grads = grad_logp.contiguous().view(-1)
        dhidden = torch.empty_like(rows)
        da = torch.zeros(lora_a.shape, dtype=torch.float32, device=hidden.device)
        db = torch.zeros(lora_b.shape, dtype=torch.float32, device=hidden.device)
        for part in _chunks(rows.shape[0], ctx.chunk_tokens):
            logits = torch.matmul(rows[part], weight.t())
            _, shrunk = sampler._lora_linear(logits, rows[part], lora_a, lora_b, adapters[part], scaling, inplace=True,
                                             return_shrunk=True)
            logp = sampler._compute_logp(logits, tokens[part])
            dlogits = sampler._compute_logp_backward(logits, tokens[part], logp, grads[part], inplace=True)
            dhidden[part], da_part, db_part = sampler._lora_linear_backward(
                dlogits, rows[part], lora_a, lora_b, adapters[part], scaling, shrunk,
                torch.matmul(dlogits, weight) if ctx.needs_input_grad[1] else None)
            da += da_part
            db += db_part
            del logits, dlogits
        needs = ctx.needs_input_grad
        return (None, dhidden.view(hidden.shape) if needs[1] else None, None, da.to(lora_a.dtype) if needs[3] else None,
                db.to(lora_b.dtype) if needs[4] else None, None, None, None, None)


def _lora_rows(hidden, token_ids, adapter_ids):
    return (hidden.contiguous().view(-1, hidden.shape[-1]), token_ids.contiguous().view(-1),
            adapter_ids.contiguous().view(-1))


def _chunks(n_rows, chunk_tokens):
    chunk = _chunk_rows(chunk_tokens, LMHEAD_BACKWARD_CHUNK_TOKENS)
    return [slice(start, min(start + chunk, n_rows)) for start in range(0, n_rows, chunk)]


def _no_gradient(scaling):
    if isinstance(scaling, torch.Tensor) and scaling.requires_grad:
        raise ValueError("there is no gradient for scaling: pass it detached")


def lora_linear(sampler, base: torch.Tensor, hidden: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                adapter_ids: torch.Tensor, scaling=1.0) -> torch.Tensor:
    """``SamplerBackend.lora_linear`` as a node of the autograd graph: gradients flow to ``base`` (the incoming one),
    ``hidden``, ``lora_a`` and ``lora_b``; not to ``scaling``.  Not differentiable twice.

    ``out = lora_linear(sampler, F.linear(hidden, weight), hidden, lora_a, lora_b, adapter_ids)``
    """
    _no_gradient(scaling)
    return _LoraLinear.apply(sampler, base, hidden, lora_a, lora_b, adapter_ids, scaling)


def lora_linear_logp(sampler, hidden: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                     token_ids: torch.Tensor, adapter_ids: torch.Tensor, scaling=1.0,
                     chunk_tokens: int | None = None) -> torch.Tensor:
    """Log-probabilities of tokens under a frozen lm_head with adapters: ``log_softmax(hidden @ weight.T + adapter)``, fp32
    of shape hidden.shape[:-1], with gradients for ``hidden``, ``lora_a`` and ``lora_b``.

    hidden: [.., H], weight: [V, H], lora_a: [S, R, H], lora_b: [S, V, R], all bf16 or all fp16; token_ids and
    adapter_ids: integers of shape hidden.shape[:-1].  Both passes hold one chunk of ``chunk_tokens`` rows of
    logits at a time; the backward builds them again.
    """
    _no_gradient(scaling)
    if weight.requires_grad:
        raise ValueError("the shared weight is frozen here: pass it detached (linear_logp has its gradient)")
    lead = tuple(hidden.shape[:-1])
    if weight.dim() != 2 or weight.shape[1] != hidden.shape[-1] or weight.shape[0] != lora_b.shape[1]:
        raise ValueError(f"weight {tuple(weight.shape)} does not fit hidden {tuple(hidden.shape)} and lora_b {tuple(lora_b.shape)}")
    _require_gpu(weight, "weight")
    if weight.dtype != hidden.dtype or weight.device != hidden.device:
        raise TypeError(f"weight is {weight.dtype} on {weight.device}, hidden {hidden.dtype} on {hidden.device}")
    if tuple(token_ids.shape) != lead or tuple(adapter_ids.shape) != lead:
        raise ValueError("token_ids and adapter_ids must have shape hidden.shape[:-1]")
    _chunk_rows(chunk_tokens, LMHEAD_BACKWARD_CHUNK_TOKENS)
    sampler._check_adapters(hidden, lora_a, lora_b, adapter_ids, scaling)
    return _LoraLinearLogp.apply(sampler, hidden, weight, lora_a, lora_b, token_ids, adapter_ids, scaling, chunk_tokens)
