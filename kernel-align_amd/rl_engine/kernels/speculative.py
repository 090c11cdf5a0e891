"""Verification of drafted tokens (speculative rollouts) on hand-written gfx950 kernels.

The reference has no counterpart: its ``sample`` (rl_engine/kernels/sampling.py:39-88) draws one token per forward pass.
``SamplerBackend`` takes the operator from here.
"""
from __future__ import annotations

from functools import cached_property, lru_cache

import torch

from rl_engine.kernels import _hip
from rl_engine.kernels._launch import _on_device, _raw_stream, _require_gpu, to_rows

_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_DRAFT = 64  # KA_VERIFY_MAX_DRAFT


class SpeculativeOps:
    @cached_property
    def _verify_workspace_bytes(self):
        """The library's query, remembered by shape."""
        return lru_cache(maxsize=1024)(self._lib.ka_verify_workspace_bytes)

    @torch.inference_mode()
    def verify_draft(self, target_logits, draft_ids, uniforms=None, draft_logits=None, draft_lens=None, top_k=None,
                     top_p=None, temperature=1.0, generator=None, return_policy_logprob=False):
        """Accept or redraw drafted tokens so that the result is distributed as ``sample`` would draw it.

        target_logits: [B, K + 1, V] bf16 / fp16 / fp32 on the GPU, the target model's logits at the K drafted positions
        and the one behind them.  draft_ids: integer [B, K].  draft_logits: [B, K, V] of the same dtype, the logits the
        drafts were drawn from, or None for drafts without probabilities (looked up, or a drafter's argmax).  draft_lens:
        integer [B], the number of drafts of each request (default: K for all; what lies behind is not read).  K <= 64;
        K = 0 is ``sample``.

        Both rows of a position are taken through the same temperature -> top-k -> top-p as in ``sample`` (scalars, or [B]
        tensors of per-request values, where a top_k of 0 filters nothing): P from the target, Q from the draft (one-hot without
        draft logits).  There is one set of parameters, one dtype and one vocabulary for both models: a drafter that sampled at
        another temperature or with other filters is not described by Q exactly (scale its logits beforehand, which rounds them;
        or draft under the target's parameters).  Draft j is accepted iff ``uniforms[:, j] * Q(d) < P(d)``; the first position that
        is not is redrawn from max(P - Q, 0), and when all are accepted the position behind them is drawn from P, both by the
        inverse CDF in index order that ``uniforms[:, K]`` drives.  All of it is decided on the sampling operator's integer masses:
        the ids are a function of the request alone.  uniforms: fp32 [B, K + 1] in [0, 1) (a last one of exactly 0 costs the
        request two serial passes over a row in 128-bit integers); None takes them from ``torch.rand(generator=generator)``.
        A draft id outside [0, V) has P = 0 and is never accepted.  (A draft that Q cannot have drawn may leave no residual,
        where P = Q: the token then comes from P.)

        Returns ``(ids, accepted)``: int64 [B, K + 1] with the accepted drafts, the drawn token and -1 behind it, and int64
        [B] with the number of accepted drafts.  With ``return_policy_logprob=True`` also fp32 [B, K + 1], every emitted
        token's log-probability under the unfiltered softmax of its target row (0 behind the last): to 1e-5 what
        ``compute_logp`` returns for it.
        """
        _require_gpu(target_logits, "target_logits")
        if target_logits.dim() != 3 or target_logits.shape[1] < 1:
            raise ValueError("target_logits must be [B, K + 1, V]")
        if target_logits.dtype not in _DTYPE_CODE:
            raise TypeError(f"unsupported logits dtype {target_logits.dtype}")
        batch, k, vocab = target_logits.shape[0], target_logits.shape[1] - 1, target_logits.shape[2]
        dev = target_logits.device
        if k > MAX_DRAFT:
            raise ValueError(f"at most {MAX_DRAFT} drafted tokens per request (got {k})")
        if vocab < 1:
            raise ValueError("target_logits have an empty vocabulary")

        def whole(t, name, shape):
            if tuple(t.shape) != shape:
                raise ValueError(f"{name} shape {tuple(t.shape)} != {shape}")
            if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
                raise TypeError(f"{name} must be integers (got {t.dtype})")
            return t if t.dtype == torch.int64 and t.device == dev and t.is_contiguous() else t.to(device=dev, dtype=torch.int64).contiguous()

        ids = whole(draft_ids, "draft_ids", (batch, k))
        lens = None if draft_lens is None else whole(draft_lens, "draft_lens", (batch,))
        if draft_logits is not None:
            _require_gpu(draft_logits, "draft_logits")
            if draft_logits.device != dev:
                raise ValueError(f"draft_logits live on {draft_logits.device}, target_logits on {dev}")
            if tuple(draft_logits.shape) != (batch, k, vocab):
                raise ValueError(f"draft_logits shape {tuple(draft_logits.shape)} != {(batch, k, vocab)}")
            if draft_logits.dtype != target_logits.dtype:
                raise TypeError(f"draft_logits are {draft_logits.dtype}, target_logits {target_logits.dtype}")
        temp, temp_rows = _per_request(temperature, "temperature", batch, dev, torch.float32, 1.0, lambda v: v > 0.0,
                                       "must be > 0")
        kk, kk_rows = _per_request(top_k, "top_k", batch, dev, torch.int32, 0, lambda v: int(v) >= 1, "must be >= 1")
        kk = min(int(kk), vocab)
        pp, pp_rows = _per_request(top_p, "top_p", batch, dev, torch.float32, 1.0, lambda v: 0.0 < v <= 1.0,
                                   "must be in (0, 1]")
        if uniforms is None:
            uniforms = torch.rand(batch, k + 1, generator=generator, device=dev, dtype=torch.float32)
        else:
            if tuple(uniforms.shape) != (batch, k + 1):
                raise ValueError(f"uniforms shape {tuple(uniforms.shape)} != {(batch, k + 1)}")
            uniforms = uniforms.to(device=dev, dtype=torch.float32).contiguous()
        out = torch.empty(batch, k + 1, dtype=torch.int64, device=dev)
        accepted = torch.empty(batch, dtype=torch.int64, device=dev)
        policy = torch.empty(batch, k + 1, dtype=torch.float32, device=dev) if return_policy_logprob else None
        if batch > 0:
            target, t_strides = _rows3(target_logits)
            draft, d_strides = (None, (0, 0)) if draft_logits is None or k == 0 else _rows3(draft_logits)
            code = _DTYPE_CODE[target_logits.dtype]
            ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
            with _on_device(dev):
                ws_bytes = self._verify_workspace_bytes(code, batch, k, vocab)
                with self._scratch(ws_bytes, dev) as ws_ptr:
                    status = self._lib.ka_verify_draft(
                        code, target.data_ptr(), *t_strides, ptr(draft), *d_strides, ids.data_ptr(), ptr(lens),
                        uniforms.data_ptr(), batch, k, vocab, float(temp), ptr(temp_rows), kk, ptr(kk_rows),
                        float(pp), ptr(pp_rows), out.data_ptr(), accepted.data_ptr(), ptr(policy), ws_ptr, ws_bytes,
                        _raw_stream())
            _hip.check(status, "ka_verify_draft")
        return (out, accepted, policy) if return_policy_logprob else (out, accepted)


def _per_request(value, name, batch, dev, dtype, default, valid, rule):
    """(scalar, [B] tensor or None) of a filter parameter given as None, a number or one value per request."""
    if isinstance(value, torch.Tensor):
        if tuple(value.shape) != (batch,):
            raise ValueError(f"{name} tensor must have shape ({batch},)")
        return default, to_rows(value, dev, dtype)
    if value is None:
        return default, None
    if not valid(value):
        raise ValueError(f"{name} {rule} (got {value})")
    return value, None


def _rows3(logits):
    """A view of [B, P, V] logits with unit stride along V and steps of at least V, and its two strides in elements; copied
    only where the layout has neither."""
    b, p, v = logits.shape
    ok = logits.stride(2) == 1 or v == 1
    ok = ok and (p <= 1 or logits.stride(1) >= v) and (b <= 1 or logits.stride(0) >= v)
    if not ok:
        logits = logits.contiguous()
    return logits, (logits.stride(0), logits.stride(1))
