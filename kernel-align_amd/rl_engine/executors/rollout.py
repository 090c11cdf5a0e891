"""Rollout executor: picks the operators for the sampling phase.

Interface of the reference's rl_engine/executors/rollout.py:8-35.  The reference
is a stub that returns two backend names; here the names are those of the HIP
operators, and ``step`` runs them on a batch of next-token logits.
"""
from __future__ import annotations

from typing import Callable, Optional, Tuple

import torch

from rl_engine.kernels.registry import kernel_registry
from rl_engine.utils.logger import logger


class RolloutExecutor:
    def __init__(self, model_config: Optional[dict] = None):
        self.config = model_config or {}
        logger.info("Initializing RolloutExecutor on the HIP operators...")

    def _select_operators(self) -> Tuple[str, str]:
        """The two names the reference selects (rollout.py:17-28): the logprob operator and "attention",
        which is outside the HIP hot path and is answered with the NOT_ON_HIP_PATH name."""
        logp_be = kernel_registry.dispatch("fused_logp")
        attn_be = kernel_registry.dispatch("attention")
        logger.info_once(f"Selected Logp backend: {logp_be}")
        logger.info_once(f"Selected Attention backend: {attn_be}")
        return logp_be, attn_be

    def execute_rollout(self):
        """Same result shape as rollout.py:30-35, plus the name of the sampling operator `step` runs."""
        logp_op, attn_op = self._select_operators()
        logger.info_once(f"Starting rollout via {logp_op}...")
        return {"status": "success", "kernels": [logp_op, attn_op],
                "sampling_kernel": kernel_registry.dispatch("sampling")}

    def step(self, logits, uniforms=None):
        """One decode step: sample a token per row of `logits` [B, V] and return (ids, logprobs)."""
        sample = kernel_registry.resolve("sampling")
        # both kernels from one operator call: at small batches the host time of a call exceeds the kernels' time
        return sample(logits, top_k=self.config.get("top_k"), top_p=self.config.get("top_p"),
                      temperature=self.config.get("temperature", 1.0), uniforms=uniforms, return_policy_logprob=True)

    def generate(self, next_logits: Callable, prompt_ids, max_new_tokens: int, uniforms=None,
                 eos_id: Optional[int] = None):
        """Autoregressive rollout of a group: ``next_logits(ids [B, t]) -> [B, V]`` supplies the logits of
        the next position; each step samples with the configured filters and records the log-probability
        of the drawn token under the unfiltered distribution (what the GRPO ratio is built from).

        prompt_ids: int64 [B, T0].  uniforms: optional fp32 [max_new_tokens, B], one draw per row and step.
        Rows that have produced ``eos_id`` keep emitting it with log-probability 0.  No step synchronises
        with the host.  Returns (ids [B, T0 + max_new_tokens], logprobs fp32 [B, max_new_tokens]).
        """
        if prompt_ids.dim() != 2:
            raise ValueError("prompt_ids must be [B, T0]")
        batch, t0 = prompt_ids.shape
        if uniforms is not None and tuple(uniforms.shape) != (max_new_tokens, batch):
            raise ValueError(f"uniforms must have shape ({max_new_tokens}, {batch})")
        ids = torch.empty(batch, t0 + max_new_tokens, dtype=torch.int64, device=prompt_ids.device)
        ids[:, :t0] = prompt_ids
        logprobs = torch.zeros(batch, max_new_tokens, dtype=torch.float32, device=prompt_ids.device)
        done = torch.zeros(batch, dtype=torch.bool, device=prompt_ids.device)
        for step in range(max_new_tokens):
            logits = next_logits(ids[:, :t0 + step])
            tok, lp = self.step(logits, None if uniforms is None else uniforms[step])
            if eos_id is not None:
                tok = torch.where(done, torch.full_like(tok, eos_id), tok)
                lp = torch.where(done, torch.zeros_like(lp), lp)
                done = done | (tok == eos_id)
            ids[:, t0 + step] = tok
            logprobs[:, step] = lp
        return ids, logprobs

    def verify_step(self, target_logits, draft_ids, draft_logits=None, draft_lens=None, uniforms=None):
        """One step on drafted tokens: accept or redraw `draft_ids` [B, K] against `target_logits` [B, K + 1, V] under the
        configured filters.  Returns (ids [B, K + 1], accepted [B], logprobs [B, K + 1]); what lies behind the
        ``accepted + 1`` tokens of a row is -1 / 0."""
        verify = kernel_registry.resolve("verify_draft")
        return verify(target_logits, draft_ids, uniforms=uniforms, draft_logits=draft_logits, draft_lens=draft_lens,
                      top_k=self.config.get("top_k"), top_p=self.config.get("top_p"),
                      temperature=self.config.get("temperature", 1.0), return_policy_logprob=True)

    def generate_speculative(self, next_logits: Callable, propose: Callable, prompt_ids, max_new_tokens: int,
                             uniforms=None, eos_id: Optional[int] = None):
        """``generate`` with drafted tokens: the same distribution of rollouts in fewer passes of the target model.

        ``propose(ids, lengths) -> (draft_ids [B, K], draft_logits [B, K, V] or None)`` drafts K tokens behind the first
        ``lengths[b]`` entries of every row of ``ids``; ``next_logits(ids, lengths, draft_ids) -> [B, K + 1, V]`` is one
        pass of the target model, its logits behind those entries and behind each draft.  ``ids`` is the int64
        [B, T0 + max_new_tokens] buffer of the rollout (zeros behind a row's length); both calls get the loop's own
        tensors and must not write to them.  A row whose rollout is complete keeps taking part with no drafts.

        prompt_ids: int64 [B, T0].  uniforms: optional fp32 [max_new_tokens, B, K + 1], one slice per pass.  Rows that have
        produced ``eos_id`` are filled with it, log-probability 0, as in ``generate``.  Every pass reads one flag back
        to the host (whether a row is left).
        Returns (ids [B, T0 + max_new_tokens], logprobs fp32 [B, max_new_tokens], passes of the target model).
        """
        if prompt_ids.dim() != 2:
            raise ValueError("prompt_ids must be [B, T0]")
        batch, t0 = prompt_ids.shape
        if uniforms is not None and (uniforms.dim() != 3 or tuple(uniforms.shape[:2]) != (max_new_tokens, batch)):
            raise ValueError(f"uniforms must have shape ({max_new_tokens}, {batch}, K + 1)")
        dev = prompt_ids.device
        total = t0 + max_new_tokens
        ids = torch.zeros(batch, total + 1, dtype=torch.int64, device=dev)  # (the last column takes what is not kept)
        ids[:, :t0] = prompt_ids
        logprobs = torch.zeros(batch, max_new_tokens + 1, dtype=torch.float32, device=dev)
        new = torch.zeros(batch, dtype=torch.int64, device=dev)  # tokens produced per row
        done = torch.zeros(batch, dtype=torch.bool, device=dev)
        passes = 0
        while passes < max_new_tokens and batch > 0 and not bool(done.all()):
            draft_ids, draft_logits = propose(ids[:, :total], t0 + new)
            k = draft_ids.shape[1]
            logits = next_logits(ids[:, :total], t0 + new, draft_ids)
            room = torch.where(done, torch.zeros_like(new), max_new_tokens - new)
            tok, accepted, lp = self.verify_step(logits, draft_ids, draft_logits, (room - 1).clamp(0, k),
                                                 None if uniforms is None else uniforms[passes])
            passes += 1
            at = torch.arange(k + 1, device=dev)
            keep = (at <= accepted[:, None]) & ~done[:, None]
            if eos_id is not None:
                ended = (tok == eos_id) & keep
                keep &= ended.cumsum(1) - ended.to(torch.int64) == 0  # up to the first end
                done = done | (ended & keep).any(1)
            where = torch.where(keep, new[:, None] + at, max_new_tokens)
            ids.scatter_(1, t0 + where, torch.where(keep, tok, torch.zeros_like(tok)))
            logprobs.scatter_(1, where, lp)
            new = new + keep.sum(1)
            done = done | (new >= max_new_tokens)
        ids, logprobs = ids[:, :total], logprobs[:, :max_new_tokens]
        if eos_id is not None:
            ids = torch.where(torch.arange(total, device=dev) < (t0 + new)[:, None], ids, torch.full_like(ids, eos_id))
        return ids.contiguous(), logprobs.contiguous(), passes
