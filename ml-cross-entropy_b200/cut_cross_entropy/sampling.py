"""Tokens from logits: temperature, top-k, top-p and min-p, drawn with given random numbers.

:func:`sample_tokens` runs ``cce_b200_sample``; :func:`linear_sample` is one decoding step of the head,
:func:`cut_cross_entropy.linear_logits` followed by it.
"""

from __future__ import annotations

import math

import torch

from . import _native
from .linear_logits import _check_device, _check_no_grad, _check_plain, _on_device, _rows, linear_logits


def _setting(name, value, batch_shape, device, dtype, hi):
    """A per-row tensor in the kernel's dtype, or the checked number for all rows: (tensor, number)."""
    if not isinstance(value, torch.Tensor):
        if not 0 <= value <= hi:  # NaN too
            raise ValueError(f"{name} must be in the range [0, {hi}]. Got {value}.")
        return None, value
    if value.shape != batch_shape:
        raise ValueError(f"Expected {name} of shape {tuple(batch_shape)}, got {tuple(value.shape)}.")
    if value.dtype != dtype:
        if value.dtype == torch.bool or value.is_complex() or (dtype == torch.int64 and value.is_floating_point()):
            raise ValueError(f"{name} of dtype {value.dtype} is not supported.")
        value = value.to(dtype)
    if value.device != device:
        raise ValueError(f"Expected {name} on {device}, got {value.device}.")
    return value.contiguous(), 0


def sample_tokens(
    logits: torch.Tensor,
    u: torch.Tensor,
    temperature: torch.Tensor | float = 1.0,
    top_k: torch.Tensor | int | None = None,
    top_p: torch.Tensor | float | None = None,
    min_p: torch.Tensor | float | None = None,
    return_logprobs: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """One token for every row of ``logits``, drawn with that row's uniform number ``u``.

    The weight of token ``v`` is ``exp((logits[v] - max) / temperature)``; a token whose logit is NaN or
    -inf, or whose weight is below ``2**-40`` (the largest is 1), is never drawn.  In order of falling logits
    (equal ones by the lower index) the shortest of three prefixes is kept: the first ``top_k``; the
    fewest whose weights reach ``top_p`` of the sum of the ``top_k``; those with a weight of at least ``min_p``.
    The first is always kept.  The token is the first kept one, by index, whose running sum of weights exceeds
    ``u`` times their sum.  The sums are exact, so equal inputs give equal tokens in every batch.

    :param logits: ``(..., V)``, bf16, fp16 or fp32; V at most 2**20, in fp32 about 780 000.
    :param u: ``(...)`` float32 in [0, 1).
    :param temperature: number or ``(...)`` tensor; 0 takes the first of the largest logits.
    :param top_k: number or ``(...)`` tensor; ``None``, 0 or V and more: off.
    :param top_p: number or ``(...)`` tensor; ``None`` or 1: off.
    :param min_p: number or ``(...)`` tensor; ``None`` or 0: off.
    :param return_logprobs: also return the logarithm of the token's share of the kept weights (float32).
    :returns: int64 tokens ``(...)``, -1 where a row has nothing to draw from (its log-probability: -inf); with
        ``return_logprobs`` the pair ``(tokens, logprobs)``.

    The numbers in tensors are not looked at on the host: there, a temperature of 0 or less (or NaN) is greedy,
    ``top_p`` outside (0, 1) and ``min_p`` outside (0, 1] act like the nearest value inside, or like "off".
    Arguments are plain tensors or parameters: DTensors and other wrappers without memory of their own are refused.
    """
    _check_plain(logits=logits, u=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    _check_no_grad("sample_tokens", logits, u, temperature, top_p, min_p)
    batch_shape = u.shape
    if logits.dim() < 1 or batch_shape != logits.shape[:-1]:
        raise ValueError(f"Expected logits (..., V) and u (...), got {tuple(logits.shape)} and {tuple(u.shape)}.")
    V = logits.size(-1)
    if V == 0:
        raise ValueError("logits have no entries.")
    if not u.is_floating_point():
        raise ValueError(f"u must be a floating-point tensor. Got {u.dtype}.")
    if isinstance(top_k, float):
        raise ValueError(f"top_k must be a whole number. Got {top_k}.")
    dev, f32 = logits.device, torch.float32
    temperature_t, temperature_n = _setting("temperature", temperature, batch_shape, dev, f32, math.inf)
    top_k_t, top_k_n = _setting("top_k", 0 if top_k is None else top_k, batch_shape, dev, torch.int64, 2**62)
    top_p_t, top_p_n = _setting("top_p", 1.0 if top_p is None else top_p, batch_shape, dev, f32, 1.0)
    min_p_t, min_p_n = _setting("min_p", 0.0 if min_p is None else min_p, batch_shape, dev, f32, 1.0)
    if not logits.is_cuda:
        raise RuntimeError("cut_cross_entropy (B200 backend) needs CUDA tensors; it has no CPU path")
    _check_device(dev, ("u", u))
    dtype = _native._DTYPE_CODE.get(logits.dtype)
    if dtype is None:
        raise NotImplementedError(
            f"logits of dtype {logits.dtype} are not supported by this backend (bf16, fp16, fp32 are)"
        )

    tokens = torch.empty(batch_shape, dtype=torch.int64, device=dev)
    logprobs = torch.empty(batch_shape, dtype=f32, device=dev) if return_logprobs else None
    with _on_device(dev):
        rows = _rows(logits, V)
        u = u.to(f32).contiguous()
        B = rows.size(0)
        args = _native.SampleArgs(
            rows.data_ptr(), B, V, rows.stride(0) if B > 1 else V, dtype, u.data_ptr(), _native._ptr(temperature_t),
            _native._ptr(top_k_t), _native._ptr(top_p_t), _native._ptr(min_p_t), temperature_n, top_p_n, min_p_n, top_k_n,
            tokens.data_ptr(), _native._ptr(logprobs),
        )  # fmt: skip
        L = _native.lib()
        ws = _native.workspace(L.cce_b200_sample_workspace_bytes(args), dev)
        rc = L.cce_b200_sample(args, ws.data_ptr(), ws.numel(), _native.stream_ptr(dev))
    if rc != 0:
        _native.check(rc, "cce_b200_sample")
    return (tokens, logprobs) if return_logprobs else tokens


def linear_sample(
    e: torch.Tensor,
    c: torch.Tensor,
    u: torch.Tensor,
    bias: torch.Tensor | None = None,
    softcap: float | None = None,
    lora_a: torch.Tensor | None = None,
    lora_b: torch.Tensor | None = None,
    adapter_ids: torch.Tensor | None = None,
    lora_scale: torch.Tensor | float | None = None,
    temperature: torch.Tensor | float = 1.0,
    top_k: torch.Tensor | int | None = None,
    top_p: torch.Tensor | float | None = None,
    min_p: torch.Tensor | float | None = None,
    return_logprobs: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """One decoding step of the head: the next token of every row of ``e``.

    ``sample_tokens(linear_logits(e, c, ..., out_dtype=torch.float32), u, ...)``; the float32 logits
    ``(..., V)`` live only during the call.  See :func:`cut_cross_entropy.linear_logits` and
    :func:`sample_tokens` for the arguments."""
    if u.shape != e.shape[:-1]:
        raise ValueError(f"Expected u of shape {tuple(e.shape[:-1])}, got {tuple(u.shape)}.")
    logits = linear_logits(
        e, c, bias=bias, softcap=softcap, lora_a=lora_a, lora_b=lora_b, adapter_ids=adapter_ids,
        lora_scale=lora_scale, out_dtype=torch.float32,
    )  # fmt: skip
    return sample_tokens(
        logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, return_logprobs=return_logprobs
    )
