"""Low-rank adapters of many requests beside a shared projection, on hand-written gfx950 kernels.

The policies of a rollout (and the policy an update trains) are adapters on one base model: the projection is shared, every
token adds its own adapter's product.  The reference has no counterpart.  ``SamplerBackend`` takes the operators from here.
"""
from __future__ import annotations

from functools import cached_property, lru_cache

import torch

from rl_engine.kernels import _hip
from rl_engine.kernels._launch import _on_device, _raw_stream, _require_gpu

_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1}
MAX_RANK = 128         # KA_LORA_MAX_RANK
MAX_ADAPTERS = 1023    # KA_LORA_MAX_ADAPTERS
MAX_TOKENS = 1 << 20   # KA_LORA_MAX_TOKENS


def _flat_rows(t):
    """[.., D] as [N, D] with unit stride along D and steps of at least D, copied only where it has no such view."""
    d = t.shape[-1]
    if t.dim() == 2 and (t.stride(1) == 1 or d == 1) and (t.shape[0] <= 1 or t.stride(0) >= d):
        return t
    return t.contiguous().view(-1, d)


def _stride(rows):
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


class AdapterOps:
    @cached_property
    def _lora_workspace_bytes(self):
        """The library's query, remembered by shape: a call of it costs as much host time as a kernel launch."""
        return lru_cache(maxsize=1024)(self._lib.ka_lora_workspace_bytes)

    def _check_adapters(self, hidden, lora_a, lora_b, adapter_ids, scaling):
        """Shapes of one call: (hidden rows, A, B, ids, scaling tensor or None, scaling number)."""
        for t, name in ((hidden, "hidden"), (lora_a, "lora_a"), (lora_b, "lora_b")):
            _require_gpu(t, name)
            if t.device != hidden.device:
                raise ValueError(f"{name} lives on {t.device}, hidden on {hidden.device}")
            if t.dtype != hidden.dtype:
                raise TypeError(f"{name} is {t.dtype}, hidden {hidden.dtype}")
        if hidden.dtype not in _DTYPE_CODE:
            raise TypeError(f"adapters take bf16 or fp16 (got {hidden.dtype})")
        if hidden.dim() < 1 or lora_a.dim() != 3 or lora_b.dim() != 3:
            raise ValueError("hidden must be [.., H], lora_a [S, R, H], lora_b [S, O, R]")
        s, r, h = lora_a.shape
        if hidden.shape[-1] != h or lora_b.shape[0] != s or lora_b.shape[2] != r:
            raise ValueError(f"hidden {tuple(hidden.shape)}, lora_a {tuple(lora_a.shape)} and lora_b {tuple(lora_b.shape)} do "
                             "not fit: they must be [.., H], [S, R, H], [S, O, R]")
        if min(s, r, h, lora_b.shape[1]) < 1:
            raise ValueError("adapters, rank and widths must be positive")
        if r > MAX_RANK:
            raise ValueError(f"rank {r} > {MAX_RANK}")
        if s > MAX_ADAPTERS:
            raise ValueError(f"{s} adapters > {MAX_ADAPTERS}")
        if tuple(adapter_ids.shape) != tuple(hidden.shape[:-1]):
            raise ValueError(f"adapter_ids shape {tuple(adapter_ids.shape)} != hidden.shape[:-1] {tuple(hidden.shape[:-1])}")
        if adapter_ids.is_floating_point() or adapter_ids.is_complex() or adapter_ids.dtype == torch.bool:
            raise TypeError(f"adapter_ids must be integers (got {adapter_ids.dtype})")
        ids = adapter_ids
        if ids.dtype != torch.int64 or ids.device != hidden.device or not ids.is_contiguous():
            ids = ids.to(device=hidden.device, dtype=torch.int64).contiguous()
        if ids.numel() > MAX_TOKENS:
            raise ValueError(f"{ids.numel()} tokens > {MAX_TOKENS}")
        if isinstance(scaling, torch.Tensor):
            if tuple(scaling.shape) != (s,):
                raise ValueError(f"scaling tensor must have shape ({s},)")
            if scaling.dtype != torch.float32 or scaling.device != hidden.device or not scaling.is_contiguous():
                scaling = scaling.to(device=hidden.device, dtype=torch.float32).contiguous()
            scale = 1.0
        else:
            scaling, scale = None, float(scaling)
        return _flat_rows(hidden), lora_a.contiguous(), lora_b.contiguous(), ids, scaling, scale

    def _launch_lora(self, base, hidden, a, b, ids, scaling, scale, out, out_stride, shrunk):
        """ka_lora_linear on checked [N, ..] rows; without `out` only the product with lora_a, into `shrunk`."""
        n, (s, r, h), o = hidden.shape[0], a.shape, b.shape[1]
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        with _on_device(hidden.device):
            ws_bytes = self._lora_workspace_bytes(n, h, o, r, s, 0)
            with self._scratch(ws_bytes, hidden.device) as ws_ptr:
                status = self._lib.ka_lora_linear(
                    _DTYPE_CODE[hidden.dtype], ptr(base), 0 if base is None else _stride(base), hidden.data_ptr(),
                    _stride(hidden), a.data_ptr(), b.data_ptr(), ids.data_ptr(), ptr(scaling), scale, ptr(out), out_stride,
                    ptr(shrunk), n, h, o, r, s, ws_ptr, ws_bytes, _raw_stream())
        _hip.check(status, "ka_lora_linear")

    @torch.inference_mode()
    def lora_linear(self, base, hidden, lora_a, lora_b, adapter_ids, scaling=1.0, inplace=False, return_shrunk=False):
        return self._lora_linear(base, hidden, lora_a, lora_b, adapter_ids, scaling, inplace, return_shrunk)

    def _lora_linear(self, base, hidden, lora_a, lora_b, adapter_ids, scaling=1.0, inplace=False, return_shrunk=False):
        """Add each token's adapter to the output of a shared projection.

        ``out[n] = base[n] + scaling[a] * (hidden[n] @ lora_a[a].T) @ lora_b[a].T`` with ``a = adapter_ids[n]``; a token whose
        id lies outside [0, S) has no adapter and keeps ``base[n]``.

        base: [.., O], the projection's output (``F.linear(hidden, weight)``); hidden: [.., H]; lora_a: [S, R, H]; lora_b:
        [S, O, R]; all bf16 or all fp16, R <= 128, S <= 1023.  adapter_ids: integer tensor of shape hidden.shape[:-1], in any
        order; scaling: a number or one per adapter ([S]).  Accumulates in fp32 and rounds once, when the sum is written.
        Infinities and NaN come out as the formula gives them.
        With ``inplace=True`` the result overwrites ``base`` (whose rows must be views of one [N, O] layout, and which must not
        be a leaf that requires grad); autograd sees that as it does torch's in-place operators, and a backward that needs the
        overwritten values raises.  With ``return_shrunk=True`` the result is ``(out, shrunk)``, shrunk fp32 [.., R] the scaled product with lora_a, which
        ``lora_linear_backward`` takes.
        """
        _require_gpu(base, "base")
        rows, a, b, ids, scaling, scale = self._check_adapters(hidden, lora_a, lora_b, adapter_ids, scaling)
        if base.device != hidden.device or base.dtype != hidden.dtype:
            raise TypeError(f"base is {base.dtype} on {base.device}, hidden {hidden.dtype} on {hidden.device}")
        s, r, h = a.shape
        o = b.shape[1]
        lead = tuple(hidden.shape[:-1])
        if tuple(base.shape) != lead + (o,):
            raise ValueError(f"base shape {tuple(base.shape)} != {lead + (o,)}")
        base_rows = _flat_rows(base)
        if inplace and base_rows.data_ptr() != base.data_ptr():
            raise ValueError("inplace=True needs base as rows of one [N, O] layout")
        if inplace and base.requires_grad and (base.is_leaf or (base._is_view() and base._base.is_leaf)):
            raise ValueError("inplace=True cannot overwrite a leaf that requires grad, or a view of one: pass it detached")
        n = rows.shape[0]
        out = base if inplace else torch.empty(lead + (o,), dtype=base.dtype, device=base.device)
        shrunk = torch.empty(lead + (r,), dtype=torch.float32, device=base.device) if return_shrunk else None
        if n > 0:
            if inplace and not base.is_inference():
                torch.autograd.graph.increment_version(base)  # the kernel writes through a pointer, which autograd does not see
            self._launch_lora(base_rows, rows, a, b, ids, scaling, scale, out, _stride(base_rows) if inplace else o, shrunk)
        return (out, shrunk) if return_shrunk else out

    @torch.inference_mode()
    def lora_linear_backward(self, grad_out, hidden, lora_a, lora_b, adapter_ids, scaling=1.0, shrunk=None,
                             dhidden_base=None):
        return self._lora_linear_backward(grad_out, hidden, lora_a, lora_b, adapter_ids, scaling, shrunk, dhidden_base)

    def _lora_linear_backward(self, grad_out, hidden, lora_a, lora_b, adapter_ids, scaling=1.0, shrunk=None,
                              dhidden_base=None):
        """Gradients of ``lora_linear`` with respect to hidden, lora_a and lora_b.

        ``grad_out`` [.., O] is also the gradient of ``base``.  ``shrunk`` is the forward's (``return_shrunk=True``); None
        computes it again.  ``dhidden_base`` [.., H], the shared projection's own gradient of hidden
        (``grad_out @ weight``), is added to the adapters' part before the sum is rounded.
        Returns ``(dhidden [.., H] in hidden's dtype, dlora_a [S, R, H] fp32, dlora_b [S, O, R] fp32)``: sums over the tokens in
        fp32 in a fixed order, zeros for an adapter without tokens.
        """
        _require_gpu(grad_out, "grad_out")
        rows, a, b, ids, scaling, scale = self._check_adapters(hidden, lora_a, lora_b, adapter_ids, scaling)
        s, r, h = a.shape
        o = b.shape[1]
        lead = tuple(hidden.shape[:-1])
        for t, name, width in ((grad_out, "grad_out", o), (dhidden_base, "dhidden_base", h)):
            if t is None:
                continue
            _require_gpu(t, name)
            if tuple(t.shape) != lead + (width,):
                raise ValueError(f"{name} shape {tuple(t.shape)} != {lead + (width,)}")
            if t.device != hidden.device or t.dtype != hidden.dtype:
                raise TypeError(f"{name} is {t.dtype} on {t.device}, hidden {hidden.dtype} on {hidden.device}")
        n = rows.shape[0]
        dev = hidden.device
        if shrunk is not None:
            _require_gpu(shrunk, "shrunk")
            if tuple(shrunk.shape) != lead + (r,):
                raise ValueError(f"shrunk shape {tuple(shrunk.shape)} != {lead + (r,)}")
            if shrunk.dtype != torch.float32 or shrunk.device != dev:
                raise TypeError(f"shrunk must be fp32 on {dev}")
            u = shrunk.contiguous()
        if n == 0:
            return (torch.zeros(lead + (h,), dtype=hidden.dtype, device=dev), torch.zeros_like(a, dtype=torch.float32),
                    torch.zeros_like(b, dtype=torch.float32))
        dy = _flat_rows(grad_out)
        if shrunk is None:
            u = torch.empty(n, r, dtype=torch.float32, device=dev)
            self._launch_lora(None, rows, a, b, ids, scaling, scale, None, 0, u)
        dx_base = None if dhidden_base is None else _flat_rows(dhidden_base)
        dx = torch.empty(lead + (h,), dtype=hidden.dtype, device=dev)
        da = torch.empty(s, r, h, dtype=torch.float32, device=dev)
        db = torch.empty(s, o, r, dtype=torch.float32, device=dev)
        with _on_device(dev):
            ws_bytes = self._lora_workspace_bytes(n, h, o, r, s, 1)
            with self._scratch(ws_bytes, dev) as ws_ptr:
                status = self._lib.ka_lora_linear_backward(
                    _DTYPE_CODE[hidden.dtype], dy.data_ptr(), _stride(dy), rows.data_ptr(), _stride(rows), a.data_ptr(),
                    b.data_ptr(), ids.data_ptr(), None if scaling is None else scaling.data_ptr(), scale, u.data_ptr(),
                    None if dx_base is None else dx_base.data_ptr(), 0 if dx_base is None else _stride(dx_base),
                    dx.data_ptr(), h, da.data_ptr(), db.data_ptr(), n, h, o, r, s, ws_ptr, ws_bytes, _raw_stream())
        _hip.check(status, "ka_lora_linear_backward")
        return dx, da, db
