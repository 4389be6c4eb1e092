"""Float64 CPU restatement of the head's serving operators, from their definitions.

``linear_logits``: softcap(e c^T + bias + the adapter of each token); ``sample_tokens``: one row at a time,
the shortest of three prefixes of the sorted row, then the running sum in order of the vocabulary.
"""

from __future__ import annotations

import math

import torch

WEIGHT_FLOOR = 2.0**-40


def linear_logits(e, c, bias=None, softcap=None, lora_a=None, lora_b=None, adapter_ids=None, lora_scale=None):
    """Returns (logits, magnitude): the sum of the absolute values of every product, which bounds rounding."""
    D, V = e.size(-1), c.size(0)
    shape = e.shape[:-1]
    e, c = e.double().reshape(-1, D), c.double()
    x, mag = e @ c.T, e.abs() @ c.abs().T
    if bias is not None:
        x, mag = x + bias.double(), mag + bias.double().abs()
    if lora_a is not None:
        for t, a in enumerate(adapter_ids.reshape(-1).tolist()):
            if 0 <= a < lora_a.size(0):
                s = 1.0 if lora_scale is None else float(lora_scale[a])
                A, B = lora_a[a].double(), lora_b[a].double()
                x[t] += s * (B @ (A @ e[t]))
                mag[t] += abs(s) * (B.abs() @ (A.abs() @ e[t].abs()))
    if softcap is not None:
        x = softcap * torch.tanh(x / softcap)
    return x.reshape(*shape, V), mag.reshape(*shape, V)


def sample_row(x, u, temperature=1.0, top_k=None, top_p=None, min_p=None) -> tuple[int, float]:
    x = x.double()
    ids = (x > -math.inf).nonzero().squeeze(1)
    if ids.numel() == 0:
        return -1, -math.inf
    x = x[ids]
    peak = x.max()
    if not temperature > 0:
        return int(ids[int((x == peak).nonzero()[0])]), 0.0
    w = torch.where(x == peak, torch.ones_like(x), torch.exp((x - peak) / temperature))
    ids, x, w = (t[w >= WEIGHT_FLOOR] for t in (ids, x, w))
    order = torch.sort(x, descending=True, stable=True).indices
    cum = w[order].cumsum(0)
    n = len(order)
    if top_k is not None and 0 < top_k < n:
        n = int(top_k)
    kept = n
    if top_p is not None and top_p < 1:
        kept = min(kept, int((cum[:n] < top_p * cum[n - 1]).sum()) + 1)
    if min_p is not None and min_p > 0:
        kept = min(kept, max(1, int((w >= min(min_p, 1.0)).sum())))
    keep = order[:kept].sort().values
    cum = w[keep].cumsum(0)
    i = min(int((cum <= u * cum[-1]).sum()), kept - 1)
    return int(ids[keep[i]]), math.log(float(w[keep[i]] / cum[-1]))


def sample_tokens(logits, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """(tokens, log-probabilities) of ``(B, V)`` logits; the settings are numbers or ``(B,)`` tensors."""
    at = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else v
    out = [
        sample_row(row, u[i].item(), at(temperature, i), at(top_k, i), at(top_p, i), at(min_p, i))
        for i, row in enumerate(logits)
    ]
    return torch.tensor([o[0] for o in out]), torch.tensor([o[1] for o in out], dtype=torch.float64)
