"""Logits of the classifier, with the low-rank adapters of many requests beside it.

``linear_cross_entropy`` trains the head without forming its logits; :func:`linear_logits` is the same
head (same ``e``, ``c``, ``bias``, ``softcap``) when it has to answer.  The work is done by
``cce_b200_logits``.
"""

from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from . import _native
from .linear_cross_entropy import _reject_dtensors

MAX_RANK = 256  # CCE_B200_MAX_RANK


def _check_plain(**named: torch.Tensor | float | None) -> None:
    """Refuses DTensors and other wrappers: they have no memory of their own, and the C interface reads their null
    pointer as "not given"."""
    for name, t in named.items():
        if type(t) is not torch.Tensor and type(t) is not torch.nn.Parameter and isinstance(t, torch.Tensor):
            _reject_dtensors(**{name: t})
            if t.numel() > 0 and t.data_ptr() == 0:
                raise ValueError(f"{name} is a {type(t).__name__}, which has no memory of its own: pass a plain tensor.")


def _check_no_grad(name: str, *tensors: torch.Tensor | float | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or torch.inference_mode().")
    if forward_ad._current_level >= 0:  # inside a dual_level; torch.no_grad() does not drop tangents
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative: pass the primal, or call it under torch.inference_mode().")


def _check_device(device: torch.device, *named: tuple[str, torch.Tensor | None]) -> None:
    for name, t in named:
        if t is not None and t.device != device:
            raise ValueError(f"Expected {name} on {device}, got {t.device}.")


def _on_device(device: torch.device):
    """A context with ``device`` as the current one; nothing to do (and to pay for) when it already is."""
    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` as ``(rows, width)`` with unit column stride and rows that do not overlap; copied only if it is not."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    s0, s1 = t.stride()
    if width == 1 and s1 != 1:  # the stride of one column says nothing
        t, s1 = t.reshape(-1).unsqueeze(1), 1
    if s1 != 1 or (t.size(0) > 1 and s0 < width):
        t = t.contiguous()
    return t


def linear_logits(
    e: torch.Tensor,
    c: torch.Tensor,
    bias: torch.Tensor | None = None,
    softcap: float | None = None,
    lora_a: torch.Tensor | None = None,
    lora_b: torch.Tensor | None = None,
    adapter_ids: torch.Tensor | None = None,
    lora_scale: torch.Tensor | float | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``softcap(e @ c.T + bias + adapters)``, where every token adds its own request's low-rank adapter.

    With ``a = adapter_ids[t]``, token ``t`` adds ``lora_scale[a] * (e[t] @ lora_a[a].T) @ lora_b[a].T``.
    No gradient is computed: inputs that require one are refused unless gradients are switched off, and inputs with a
    forward-mode tangent are refused.
    Arguments are plain tensors or parameters: DTensors and other wrappers without memory of their own are refused.

    :param e: embeddings ``(..., D)``: bf16, fp16, or fp32 (computed as a three-term bf16 split:
        about 16 mantissa bits; infinite entries of ``e`` or ``c`` give NaN).
    :param c: classifier ``(V, D)`` of the same dtype.
    :param bias: optional ``(V,)``, bf16, fp16 or fp32.
    :param softcap: if set, logits become ``softcap * tanh(logits / softcap)``.
    :param lora_a: ``(n_adapters, rank, D)`` in the dtype of ``e``, rank at most 256; adapters of a
        smaller rank are padded with zeros.  Given together with ``lora_b`` and ``adapter_ids``, or not at all.
    :param lora_b: ``(n_adapters, V, rank)`` in the dtype of ``e``.
    :param adapter_ids: ``(...)``, int32 or int64: the adapter of every token; -1 (or any number that names no
        adapter) for none.
    :param lora_scale: ``(n_adapters,)`` or one number for all; 1 if not given.
    :param out_dtype: bf16, fp16 or fp32; the dtype of ``e`` if not given.
    :returns: ``(..., V)``.

    Under autocast ``e``, ``c`` and the adapters are cast to the autocast dtype first.
    """
    _check_plain(e=e, c=c, bias=bias, lora_a=lora_a, lora_b=lora_b, adapter_ids=adapter_ids, lora_scale=lora_scale)
    _check_no_grad("linear_logits", e, c, bias, lora_a, lora_b, lora_scale)
    if e.dim() < 1 or c.dim() != 2 or e.size(-1) != c.size(1):
        raise ValueError(f"Expected e (..., D) and c (V, D), got {tuple(e.shape)} and {tuple(c.shape)}.")
    if bias is not None and bias.shape != c.shape[:1]:
        raise ValueError(f"Expected bias of shape {tuple(c.shape[:1])}, got {tuple(bias.shape)}.")
    if softcap is not None and not softcap > 0:
        raise ValueError(f"softcap must be positive. Got {softcap}.")
    given = [t is not None for t in (lora_a, lora_b, adapter_ids)]
    if any(given) != all(given):
        raise ValueError("lora_a, lora_b and adapter_ids are given together or not at all.")
    if lora_a is not None:
        if lora_a.dim() != 3 or lora_a.size(0) < 1 or not 1 <= lora_a.size(1) <= MAX_RANK:
            raise ValueError(f"Expected lora_a (n, rank <= {MAX_RANK}, D), got {tuple(lora_a.shape)}.")
        n, rank = lora_a.shape[:2]
        if lora_a.size(2) != e.size(-1) or lora_b.shape != (n, c.size(0), rank):
            raise ValueError(
                f"Expected lora_a {(n, rank, e.size(-1))} and lora_b {(n, c.size(0), rank)}, "
                f"got {tuple(lora_a.shape)} and {tuple(lora_b.shape)}."
            )
        if adapter_ids.shape != e.shape[:-1]:
            raise ValueError(f"Expected adapter_ids of shape {tuple(e.shape[:-1])}, got {tuple(adapter_ids.shape)}.")
        if adapter_ids.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"adapter_ids must be int32 or int64. Got {adapter_ids.dtype}.")
        if isinstance(lora_scale, torch.Tensor) and lora_scale.shape != (n,):
            raise ValueError(f"Expected lora_scale of shape {(n,)}, got {tuple(lora_scale.shape)}.")
    elif lora_scale is not None:
        raise ValueError("lora_scale is given without adapters.")
    if not e.is_cuda:
        raise RuntimeError("cut_cross_entropy (B200 backend) needs CUDA tensors; it has no CPU path")
    scale_t = lora_scale if isinstance(lora_scale, torch.Tensor) else None
    _check_device(e.device, ("c", c), ("bias", bias), ("lora_a", lora_a), ("lora_b", lora_b),
                  ("adapter_ids", adapter_ids), ("lora_scale", scale_t))  # fmt: skip

    if torch.is_autocast_enabled("cuda"):
        amp_dtype = torch.get_autocast_dtype("cuda")
        e, c = e.to(amp_dtype), c.to(amp_dtype)
        if lora_a is not None:
            lora_a, lora_b = lora_a.to(amp_dtype), lora_b.to(amp_dtype)
    dtype = e.dtype
    for name, t in (("c", c), ("lora_a", lora_a), ("lora_b", lora_b)):
        if t is not None and t.dtype != dtype:
            raise ValueError(f"Expected {name} in the dtype of e, {dtype}, got {t.dtype}.")
    out_dtype = dtype if out_dtype is None else out_dtype
    for what, d in (("e", dtype), ("bias", dtype if bias is None else bias.dtype), ("out", out_dtype)):
        if d not in _native._DTYPE_CODE:
            raise NotImplementedError(f"{what} of dtype {d} is not supported by this backend (bf16, fp16, fp32 are)")

    D, V = e.size(-1), c.size(0)
    out = torch.empty((*e.shape[:-1], V), dtype=out_dtype, device=e.device)
    if out.numel() == 0:
        return out
    with _on_device(e.device):
        e, c = _rows(e, D), _rows(c, D)
        bias = None if bias is None else bias.contiguous()
        args = _native.LogitsArgs()
        args.op = _native.make_operands(e, c, bias, None, softcap)
        args.out, args.out_dtype = out.data_ptr(), _native._DTYPE_CODE[out_dtype]
        if lora_a is not None:
            lora_a, lora_b, ids = lora_a.contiguous(), lora_b.contiguous(), adapter_ids.contiguous()
            args.lora_a, args.lora_b, args.adapter_ids = lora_a.data_ptr(), lora_b.data_ptr(), ids.data_ptr()
            args.ids_dtype = _native.IDX_I64 if ids.dtype == torch.int64 else _native.IDX_I32
            args.n_adapters, args.rank = n, rank
            if lora_scale is not None:
                if scale_t is None:
                    scale_t = torch.full((n,), float(lora_scale), device=e.device)
                scale_t = scale_t.to(torch.float32).contiguous()
                args.lora_scale = scale_t.data_ptr()
        L = _native.lib()
        ws = _native.workspace(L.cce_b200_logits_workspace_bytes(args), e.device)
        rc = L.cce_b200_logits(args, ws.data_ptr(), ws.numel(), _native.stream_ptr(e.device))
    if rc != 0:
        _native.check(rc, "cce_b200_logits")
    _native.finish(ws, "cce_b200_logits")
    return out
