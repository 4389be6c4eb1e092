"""Timed cases of the head's serving operators: logits with adapters, and sampling from logits.

``linear_logits``  softcap(e c^T + bias + the low-rank adapter of each token's request)
``sample_tokens``  one token per row of logits, by temperature, top-k, top-p and min-p, from given
                   uniform numbers, with the log-probability of the token

``run`` computes them in plain torch operations while ``own`` is false, and through
``cut_cross_entropy`` while it is true.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# A token whose weight is below this share of the likeliest one's is never drawn.
_WEIGHT_FLOOR = 2.0**-40


def _logits_case(name, tokens, vocab, hidden, dtype, out, adapters, rank, layout, bias=False, softcap=0.0):
    return dict(name=name, op="logits", tokens=tokens, vocab=vocab, hidden=hidden, dtype=dtype, out=out,
                adapters=adapters, rank=rank, layout=layout, bias=bias, softcap=softcap)  # fmt: skip


def _sample_case(name, rows, vocab, dtype, filters, masked=False):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, dtype=dtype, filters=filters, masked=masked)


def listed():
    return [
        # one request that decodes: the latency of a single token through the whole classifier
        _logits_case("logits_1tok_128k", 1, 128256, 4096, "bf16", "bf16", 4, 16, "each"),
        # a decode batch without adapters: the classifier is read once for eight tokens
        _logits_case("logits_8tok_256k_plain", 8, 256000, 2304, "bf16", "fp32", 0, 0, "none"),
        # a decode batch whose requests use different adapters, soft-capped, on the way to sampling
        _logits_case("logits_32tok_256k_cap", 32, 256000, 2304, "bf16", "fp32", 8, 16, "each", softcap=30.0),
        # a larger batch with some tokens of each request (draft tokens that are verified), with a bias
        _logits_case("logits_200tok_152k_fp16", 200, 152064, 3584, "fp16", "fp16", 12, 32, "runs", bias=True),
        # whole prompts scored at once: few adapters, many tokens each
        _logits_case("logits_2048tok_128k", 2048, 128256, 4096, "bf16", "bf16", 4, 64, "runs"),
        # a small head of odd sizes, whose rows no 16-byte load can address
        _logits_case("logits_37tok_odd", 37, 5003, 1001, "bf16", "bf16", 3, 8, "each", bias=True),
        # one request: latency
        _sample_case("sample_1x256k_all", 1, 256000, "fp32", "all"),
        # a decode batch with every row's own settings
        _sample_case("sample_64x128k_kp_bf16", 64, 128256, "bf16", "kp"),
        # a large batch with nucleus sampling
        _sample_case("sample_512x152k_p", 512, 152064, "fp32", "p"),
        # rollouts at a temperature, nothing cut off
        _sample_case("sample_256x256k_none", 256, 256000, "fp32", "none"),
        # the usual top-k of a small batch
        _sample_case("sample_8x128k_k", 8, 128256, "fp32", "k"),
        # a small odd vocabulary under a grammar's mask
        _sample_case("sample_33x32003_fp16_masked", 33, 32003, "fp16", "all", masked=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        case = dict(op="logits")
        case["tokens"] = _log_int(rng, 1, 2048)
        case["vocab"] = _log_int(rng, 4000, 256000)
        case["hidden"] = _log_int(rng, 256, 4096)
        if rng.random() < 0.7:  # most heads have a width that vector loads can address
            case["hidden"] = max(256, case["hidden"] // 64 * 64)
        # no dearer than the largest listed case
        while case["tokens"] * case["vocab"] * case["hidden"] > 2048 * 128256 * 4096:
            case["tokens"] = max(1, case["tokens"] // 2)
        case["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
        case["out"] = rng.choice([case["dtype"], "fp32"])
        case["layout"] = rng.choice(["none", "each", "runs", "runs"])
        case["adapters"] = 0 if case["layout"] == "none" else rng.randint(1, 16)
        case["rank"] = 0 if case["layout"] == "none" else rng.choice([4, 8, 16, 24, 32, 64])
        case["bias"] = rng.random() < 0.4
        case["softcap"] = 30.0 if rng.random() < 0.3 else 0.0
        return case
    case = dict(op="sample")
    case["vocab"] = _log_int(rng, 4000, 256000)
    case["rows"] = min(_log_int(rng, 1, 512), 512 * 152064 // case["vocab"])
    case["dtype"] = rng.choice(["fp32", "bf16", "fp16"])
    case["filters"] = rng.choice(["none", "k", "p", "kp", "all"])
    case["masked"] = rng.random() < 0.3
    return case


def _prepare_logits(case, gen):
    T, V, D = case["tokens"], case["vocab"], case["hidden"]
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    state = dict(op="logits", e=normal(T, D), c=normal(V, D, std=2.5 / D**0.5), bias=None, softcap=None,
                 lora_a=None, lora_b=None, adapter_ids=None, lora_scale=None, out_dtype=_DTYPES[case["out"]])  # fmt: skip
    if case["bias"]:
        state["bias"] = torch.randn(V, generator=gen, device="cuda") * 0.1
    if case["softcap"]:
        state["softcap"] = case["softcap"]
    if case["adapters"]:
        n, r = case["adapters"], case["rank"]
        state["lora_a"] = normal(n, r, D, std=1.0 / D**0.5)
        state["lora_b"] = normal(n, V, r, std=0.5 / r**0.5)
        state["lora_scale"] = torch.rand(n, generator=gen, device="cuda") * 1.5 + 0.5
        # -1: a request without an adapter
        if case["layout"] == "each":
            state["adapter_ids"] = torch.randint(-1, n, (T,), generator=gen, device="cuda")
        else:  # runs of tokens of one request
            length = max(1, T // (2 * n))
            starts = torch.randint(0, length, (T,), generator=gen, device="cuda") == 0
            runs = torch.cumsum(starts, 0)
            state["adapter_ids"] = torch.randint(-1, n, (T + 1,), generator=gen, device="cuda")[runs]
    return state


def _prepare_sample(case, gen):
    B, V = case["rows"], case["vocab"]

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    logits = torch.randn(B, V, generator=gen, device="cuda") * 2.5
    # a handful of likely tokens in every row, more or less sure of itself
    likely = torch.randint(0, V, (B, 40), generator=gen, device="cuda")
    logits.scatter_add_(1, likely, uniform(B, 1) * 14.0 * uniform(B, 40))
    if case["masked"]:
        logits.masked_fill_(uniform(B, V) < 0.9, -math.inf)
    filters = case["filters"]
    state = dict(op="sample", logits=logits.to(_DTYPES[case["dtype"]]), u=uniform(B), top_k=None, top_p=None,
                 min_p=None, temperature=0.3 + 1.2 * uniform(B))  # fmt: skip
    if filters == "all":  # a few greedy rows among the others
        state["temperature"] = torch.where(uniform(B) < 0.1, torch.zeros(B, device="cuda"), state["temperature"])
        state["min_p"] = 0.2 * uniform(B) * (uniform(B) < 0.7)
    if filters in ("k", "kp", "all"):
        state["top_k"] = torch.exp(uniform(B) * math.log(1000.0)).round().to(torch.int64)
    if filters in ("p", "kp", "all"):
        state["top_p"] = 0.5 + 0.49 * uniform(B)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_logits(case, gen) if case["op"] == "logits" else _prepare_sample(case, gen)


def _plain_logits(s):
    e = s["e"].float()
    x = e @ s["c"].float().t()
    if s["bias"] is not None:
        x += s["bias"].float()
    if s["lora_a"] is not None:
        for a in range(s["lora_a"].size(0)):
            h = (e @ s["lora_a"][a].float().t()) * s["lora_scale"][a]
            h = torch.where((s["adapter_ids"] == a)[:, None], h, torch.zeros_like(h))
            x += h @ s["lora_b"][a].float().t()
    if s["softcap"] is not None:
        x = torch.tanh(x / s["softcap"]) * s["softcap"]
    return x.to(s["out_dtype"])


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top, best = x.sort(dim=1, descending=True, stable=True)  # ties: the lowest index first
    peak = top[:, :1]
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    # weights in order of likelihood; equal to the peak counts as 1 even where the peak is infinite
    w = torch.where(top == peak, torch.ones_like(top), torch.exp((top - peak) / torch.where(greedy, 1.0, t)))
    w = torch.where(w < _WEIGHT_FLOOR, torch.zeros_like(w), w)
    place = torch.arange(V, device=x.device)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        w = torch.where((place < k) | (k <= 0), w, torch.zeros_like(w))
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_p"] is not None:
        cum = torch.cumsum(w, 1)
        before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
        p = s["top_p"].double()[:, None]
        keep &= (before < p * cum[:, -1:]) | (p >= 1) | (place == 0)
    if s["min_p"] is not None:
        keep &= (w >= s["min_p"].double()[:, None]) | (place == 0)
    keep &= ~greedy | (place == 0)
    w = torch.where(keep, w, torch.zeros_like(w))
    # drawn in order of the vocabulary
    w = torch.zeros_like(w).scatter_(1, best, w)
    cum = torch.cumsum(w, 1)
    total = cum[:, -1:]
    token = (cum <= s["u"].double()[:, None] * total).sum(1).clamp_(max=V - 1)
    logp = torch.log(w.gather(1, token[:, None]) / total).squeeze(1)
    none = torch.isneginf(peak).squeeze(1)  # every token masked
    token = torch.where(none, torch.full_like(token, -1), token)
    logp = torch.where(none, torch.full_like(logp, -math.inf), logp)
    return token, logp.float()


def run(state):
    if not own:
        return _plain_logits(state) if state["op"] == "logits" else _plain_sample(state)
    cce = _package()
    if state["op"] == "logits":
        return cce.linear_logits(
            state["e"], state["c"], bias=state["bias"], softcap=state["softcap"], lora_a=state["lora_a"],
            lora_b=state["lora_b"], adapter_ids=state["adapter_ids"], lora_scale=state["lora_scale"],
            out_dtype=state["out_dtype"],
        )  # fmt: skip
    return cce.sample_tokens(
        state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
        min_p=state["min_p"], return_logprobs=True,
    )  # fmt: skip


def _package():
    path = str(Path("ml-cross-entropy_b200").resolve())
    if path not in sys.path:
        sys.path.insert(0, path)
    import cut_cross_entropy

    return cut_cross_entropy


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "sample":
        B, V = case["rows"], case["vocab"]
        # a subtraction, a product, an exponential and a sum for every logit
        return {"bytes": B * V * size[case["dtype"]] + B * (4 + 16 + 12), "flops": 4 * B * V}
    T, V, D, r = case["tokens"], case["vocab"], case["hidden"], case["rank"]
    b = size[case["dtype"]]
    used = min(case["adapters"], T)
    n_bytes = (T * D + V * D + used * r * (D + V)) * b + T * V * size[case["out"]]
    n_bytes += V * 4 * case["bias"] + T * 8 * (used > 0)
    return {"bytes": n_bytes, "flops": 2 * T * V * D + (2 * T * r * (D + V) if used else 0)}


def _exact_logits(s):
    e = s["e"].double()
    V = s["c"].size(0)
    out = torch.empty(e.size(0), V, dtype=torch.float64, device=e.device)
    groups = []
    if s["lora_a"] is not None:
        for a in s["adapter_ids"].unique().tolist():
            if a >= 0:
                rows = (s["adapter_ids"] == a).nonzero().squeeze(1)
                groups.append((a, rows, torch.einsum("td,rd->tr", e[rows], s["lora_a"][a].double())))
    for v0 in range(0, V, 16384):
        v1 = min(V, v0 + 16384)
        part = torch.einsum("td,vd->tv", e, s["c"][v0:v1].double())
        if s["bias"] is not None:
            part = part + s["bias"][v0:v1].double()
        for a, rows, h in groups:
            delta = torch.einsum("tr,vr->tv", h, s["lora_b"][a, v0:v1].double())
            part[rows] += delta * s["lora_scale"][a].double()
        if s["softcap"] is not None:
            part = torch.tanh(part / s["softcap"]) * s["softcap"]
        out[:, v0:v1] = part
    return out


def _exact_row(x, u, t, k, p, m):
    """One row, from the definition: the shortest of three prefixes of the tokens in order."""
    x = x.double()
    ids = (x > -math.inf).nonzero().squeeze(1)  # NaN and -inf are masked
    if ids.numel() == 0:
        return -1, -math.inf
    x = x[ids]
    peak = x.max()
    if t <= 0:
        return int(ids[(x == peak).nonzero()[0, 0]]), 0.0
    w = torch.exp((x - peak) / t)
    w[x == peak] = 1.0
    ids, x, w = ids[w >= _WEIGHT_FLOOR], x[w >= _WEIGHT_FLOOR], w[w >= _WEIGHT_FLOOR]
    order = torch.argsort(-x, stable=True)
    cum = w[order].cumsum(0)
    n = cum.numel()
    if k is not None and k > 0:
        n = min(n, k)
    n_kept = n
    if p is not None and p < 1:
        n_kept = min(n_kept, int((cum[:n] < p * cum[n - 1]).sum()) + 1)
    if m is not None:
        n_kept = min(n_kept, max(1, int((w >= m).sum())))
    kept = order[:n_kept].sort().values
    cum = w[kept].cumsum(0)
    i = min(int((cum <= u * cum[-1]).sum()), n_kept - 1)
    return int(ids[kept[i]]), math.log(float(w[kept[i]]) / float(cum[-1]))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(s)
    per_row = [None if v is None else v.tolist() for v in (s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])]
    got = [_exact_row(row, *(None if v is None else v[i] for v in per_row)) for i, row in enumerate(s["logits"])]
    device = s["logits"].device
    return (torch.tensor([g[0] for g in got], dtype=torch.int64, device=device),
            torch.tensor([g[1] for g in got], dtype=torch.float64, device=device))  # fmt: skip
