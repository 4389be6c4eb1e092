"""Head operators on the GPU against the float64 oracle: logits with adapters, sampling, and both together."""

from __future__ import annotations

import math

import pytest
import torch

from cut_cross_entropy import _native, linear_logits, linear_sample, sample_tokens
from oracle import head_oracle as H

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


# ------------------------------------------------------------------ logits


def _tolerance(ref, mag, dtype, out_dtype, K, softcap):
    """Rounding of the result (half a step of out_dtype), fp32 accumulation of K products in any order with
    truncation (a whole step 2^-23 each), the two-step adapter product's (within the same K), for fp32 operands the
    split's dropped terms (2^-15 of every product), and the soft-cap's tanh (4 steps of 1)."""
    tol = torch.finfo(out_dtype).eps / 2 * ref.abs() + K * 2.0**-23 * mag
    if dtype == FP32:
        tol = tol + 2.0**-15 * mag
    if softcap is not None:
        tol = tol + softcap * 2.0**-21
    return tol * 1.01 + torch.finfo(out_dtype).smallest_normal


def _inputs(T, V, D, dtype, n=0, r=0, bias=None, seed=0, layout="each"):
    g = torch.Generator().manual_seed(seed)
    kw = dict(e=torch.randn(T, D, generator=g).to(dtype), c=(torch.randn(V, D, generator=g) * 2 / D**0.5).to(dtype))
    if bias is not None:
        kw["bias"] = (torch.randn(V, generator=g) * 0.3).to(bias)
    if n:
        kw["lora_a"] = (torch.randn(n, r, D, generator=g) / D**0.5).to(dtype)
        kw["lora_b"] = torch.randn(n, V, r, generator=g).to(dtype)
        kw["lora_scale"] = torch.rand(n, generator=g) + 0.5
        ids = torch.randint(-1, n, (T,), generator=g)
        kw["adapter_ids"] = ids.sort().values if layout == "runs" else ids
    return kw


def _to_dev(kw):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}


def _check_logits(kw, out_dtype=None, softcap=None):
    ref, mag = H.linear_logits(**kw, softcap=softcap)
    got = linear_logits(**_to_dev(kw), softcap=softcap, out_dtype=out_dtype)
    dtype = kw["e"].dtype
    out_dtype = out_dtype or dtype
    assert got.dtype == out_dtype and got.shape == ref.shape
    K = kw["e"].size(-1) + (kw["lora_a"].size(1) if "lora_a" in kw else 0) + 8
    err = (got.cpu().double() - ref).abs()
    assert bool((err <= _tolerance(ref, mag, dtype, out_dtype, K, softcap)).all()), err.max()
    return got


@pytest.mark.parametrize("T", [1, 2, 16, 17, 31, 33, 64, 100, 255, 256, 257, 300, 520])
def test_logits_token_counts(T):
    _check_logits(_inputs(T, 384, 192, BF16, n=3, r=16, seed=T), out_dtype=FP32)


@pytest.mark.parametrize("V", [1, 7, 127, 128, 129, 1000, 19077])
@pytest.mark.parametrize("D", [1, 8, 63, 64, 200, 1001])
def test_logits_sizes(V, D):
    _check_logits(_inputs(5, V, D, BF16, n=2, r=8, bias=FP32, seed=V + D))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("out_dtype", [None, BF16, FP16, FP32])
@pytest.mark.parametrize("bias", [None, BF16, FP16, FP32])
def test_logits_types(dtype, out_dtype, bias):
    _check_logits(_inputs(37, 300, 136, dtype, n=2, r=12, bias=bias), out_dtype=out_dtype, softcap=5.0)


@pytest.mark.parametrize("r", [1, 3, 4, 8, 15, 16, 17, 24, 32, 64, 100, 256])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_logits_ranks(r, dtype):
    _check_logits(_inputs(40, 260, 128, dtype, n=4, r=r, seed=r), out_dtype=FP32)


@pytest.mark.parametrize("n", [1, 2, 50, 300])
@pytest.mark.parametrize("layout", ["each", "runs"])
@pytest.mark.parametrize("T", [3, 290])
def test_logits_adapter_mixes(n, layout, T):
    _check_logits(_inputs(T, 200, 64, BF16, n=n, r=16, layout=layout, seed=n), out_dtype=FP32)


def test_logits_without_adapters_and_with_none_chosen():
    kw = _inputs(20, 500, 128, BF16, n=3, r=16)
    kw["adapter_ids"].fill_(-1)
    with_none = linear_logits(**_to_dev(kw), out_dtype=FP32)
    for k in ("lora_a", "lora_b", "lora_scale", "adapter_ids"):
        del kw[k]
    assert torch.equal(with_none, _check_logits(kw, out_dtype=FP32))


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_logits_ids_outside_the_adapters_mean_none(ids_dtype):
    kw = _inputs(8, 300, 64, BF16, n=2, r=8)
    kw["adapter_ids"] = torch.tensor([0, 1, 2, 100, -1, -7, 2**31 - 1, 1]).to(ids_dtype)
    _check_logits(kw, out_dtype=FP32)


def test_logits_scale_forms():
    kw = _inputs(8, 300, 64, BF16, n=2, r=8)
    kw["lora_scale"] = torch.full((2,), 0.75)
    want = linear_logits(**_to_dev(kw), out_dtype=FP32)
    assert torch.equal(linear_logits(**_to_dev(dict(kw, lora_scale=0.75)), out_dtype=FP32), want)
    kw["lora_scale"] = None
    _check_logits(kw, out_dtype=FP32)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_logits_a_broken_adapter_stays_with_its_own_requests(bad):
    kw = _inputs(48, 300, 128, BF16, n=3, r=16)
    kw["adapter_ids"] = torch.arange(48) % 4 - 1
    good = linear_logits(**_to_dev(kw), out_dtype=FP32)
    kw["lora_a"][1] = bad
    kw["lora_b"][1] = bad
    got = linear_logits(**_to_dev(kw), out_dtype=FP32)
    others = (kw["adapter_ids"] != 1).to(DEV)
    assert torch.equal(got[others], good[others])
    assert not torch.isfinite(got[~others]).any()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("r", [8, 12, 16, 40, 64, 136])
@pytest.mark.parametrize("layout", ["each", "runs"])
def test_logits_infinite_entries_of_b_give_infinities(dtype, r, layout):
    """One infinity in some rows of B, finite h: the definition's infinity, on the tensor cores (groups of one adapter)
    and in the epilogue (rank 12, fp32) alike."""
    T, V = 96, 400
    kw = _inputs(T, V, 128, dtype, n=3, r=r, seed=r, layout=layout)
    # whole numbers among the inner products, which leave nothing for a low term
    kw["lora_a"][:, 0] = 0
    kw["lora_a"][:, 0, 0] = 1
    kw["lora_scale"] = torch.ones(3)
    kw["e"][::2, 0] = torch.arange(1, T // 2 + 1).to(dtype)
    g = torch.Generator().manual_seed(r)
    rows = torch.randperm(V, generator=g)[:100]
    where = torch.randint(0, r, (100,), generator=g)
    where[:30] = 0
    kw["lora_b"][1, rows, where] = math.inf * (1 - 2 * torch.randint(0, 2, (100,), generator=g)).to(dtype)
    ref, mag = H.linear_logits(**kw)
    assert not torch.isnan(ref).any() and torch.isinf(ref).any()
    finite = torch.isfinite(ref)
    for out in (dtype, FP32):
        for t in (slice(None), slice(5, 6)):
            got = linear_logits(**_to_dev(dict(kw, e=kw["e"][t], adapter_ids=kw["adapter_ids"][t])), out_dtype=out).cpu().double()
            f = finite[t]
            assert torch.equal(got[~f], ref[t][~f])
            tol = _tolerance(ref[t], mag[t], dtype, out, 128 + r + 8, None)
            assert bool(((got - ref[t]).abs() <= tol)[f].all())


def test_logits_strides_and_shapes():
    kw = _inputs(24, 300, 128, BF16, n=2, r=16, bias=BF16)
    want = linear_logits(**_to_dev(kw), out_dtype=FP32)
    d = _to_dev(kw)
    pad = lambda x, by: torch.cat([x, torch.full((*x.shape[:-1], by), math.nan, dtype=x.dtype, device=DEV)], -1)
    for name, by in (("e", 8), ("e", 3), ("c", 16), ("c", 1), ("lora_a", 5), ("lora_b", 1)):
        view = pad(d[name], by)[..., : d[name].size(-1)]
        assert torch.equal(linear_logits(**dict(d, **{name: view}), out_dtype=FP32), want), (name, by)
    for name in ("e", "c", "lora_a", "lora_b"):  # bases off a 16-byte boundary, and transposed storage
        x = d[name]
        off = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)
        got = linear_logits(**dict(d, **{name: off}), out_dtype=FP32)
        if name == "lora_b":  # its rows are then read by the epilogue, which rounds in another order
            ref, mag = H.linear_logits(**kw)
            assert bool(((got.cpu().double() - ref).abs() <= _tolerance(ref, mag, BF16, FP32, 152, None)).all())
        else:
            assert torch.equal(got, want), name
        tr = x.transpose(-1, -2).contiguous().transpose(-1, -2)
        assert torch.equal(linear_logits(**dict(d, **{name: tr}), out_dtype=FP32), want), name
    shaped = dict(d, e=d["e"].view(2, 3, 4, 128), adapter_ids=d["adapter_ids"].view(2, 3, 4))
    assert torch.equal(linear_logits(**shaped, out_dtype=FP32), want.view(2, 3, 4, 300))
    # a token alone takes its adapter on the tensor cores, in a group of several adapters in the epilogue
    _check_logits(dict(kw, e=kw["e"][5], adapter_ids=kw["adapter_ids"][5]), out_dtype=FP32)
    same = dict(d, e=d["e"][:1].expand(24, 128))
    assert torch.equal(linear_logits(**same, out_dtype=FP32)[0], want[0])


def test_logits_empty():
    kw = _to_dev(_inputs(0, 300, 64, BF16, n=2, r=8))
    assert linear_logits(**kw).shape == (0, 300)
    kw = _to_dev(_inputs(4, 0, 64, BF16))
    assert linear_logits(**kw).shape == (4, 0)


def test_logits_refusals_on_the_device():
    kw = _to_dev(_inputs(4, 300, 64, BF16, n=2, r=8))
    with pytest.raises(ValueError):
        linear_logits(**dict(kw, c=kw["c"].half()))
    with pytest.raises(ValueError):
        linear_logits(**dict(kw, lora_a=kw["lora_a"].float()))
    with pytest.raises(ValueError):
        linear_logits(**dict(kw, adapter_ids=kw["adapter_ids"].cpu()))
    with pytest.raises(NotImplementedError):
        linear_logits(kw["e"].double(), kw["c"].double())
    with pytest.raises(NotImplementedError):
        linear_logits(kw["e"], kw["c"], out_dtype=torch.float64)


def test_logits_parameters_need_no_grad_and_autocast_casts():
    kw = _to_dev(_inputs(4, 300, 64, FP32))
    c = torch.nn.Parameter(kw["c"])
    with pytest.raises(RuntimeError):
        linear_logits(kw["e"], c)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        got = linear_logits(kw["e"], c)
    assert torch.equal(got, linear_logits(kw["e"].bfloat16(), kw["c"].bfloat16()))


def test_logits_do_not_depend_on_the_batch_mates():
    """A token's logits are the same bits alone and in a batch of any size (one order of the sums)."""
    kw = _to_dev(_inputs(300, 500, 320, BF16))
    full = linear_logits(**kw, out_dtype=FP32)
    for t in (0, 17, 255, 256, 299):
        assert torch.equal(linear_logits(**dict(kw, e=kw["e"][t : t + 1]), out_dtype=FP32)[0], full[t])
    # so they are with adapters, as long as the groups of 16 tokens stay of one adapter, or of several
    kw = _to_dev(_inputs(320, 500, 320, BF16, n=3, r=24))
    kw["adapter_ids"] = torch.arange(320, device=DEV) // 16 % 4 - 1
    full = linear_logits(**kw, out_dtype=FP32)
    for t in (0, 17, 255, 256, 319):
        one = dict(kw, e=kw["e"][t : t + 1], adapter_ids=kw["adapter_ids"][t : t + 1])
        assert torch.equal(linear_logits(**one, out_dtype=FP32)[0], full[t])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("r", [8, 16, 32, 40, 64, 72, 136, 256])
def test_logits_groups_of_one_adapter_and_mixed_ones(dtype, r):
    """Runs that start and end on and off the groups of 16 tokens, across the tiles of 256."""
    kw = _inputs(600, 300, 96, dtype, n=4, r=r, seed=r)
    ids = torch.full((600,), -1)
    for a, lo, hi in ((0, 0, 16), (1, 16, 48), (2, 50, 200), (3, 200, 300), (0, 300, 301), (1, 320, 600)):
        ids[lo:hi] = a
    kw["adapter_ids"] = ids
    for out in (dtype, FP32):
        _check_logits(kw, out_dtype=out)


@pytest.mark.parametrize("T, n", [(1024, 3), (1025, 60), (2500, 200), (9000, 1100), (300, 9000)])
def test_logits_many_tokens_and_adapters(T, n):
    """Column orders of more than one block's width of tokens and of adapters, and too many adapters for an order."""
    _check_logits(_inputs(T, 40, 64, BF16, n=n, r=8, seed=T), out_dtype=FP32)


def test_logits_inner_products_beyond_the_16_bit_type():
    """h above fp16's range: such groups take their adapter in fp32."""
    kw = _inputs(64, 300, 128, FP16, n=2, r=16)
    kw["adapter_ids"] = torch.arange(64) // 32
    kw["lora_scale"] = torch.tensor([3e5, 1.0])
    kw["lora_b"] = (kw["lora_b"].float() * 2.0**-10).half()
    ref, _ = H.linear_logits(**kw)
    assert ref.abs().max() < 60000
    _check_logits(kw, out_dtype=FP32)


@pytest.mark.parametrize("D", [64, 512, 520, 1024])
@pytest.mark.parametrize("T", [5, 100, 150, 250])
@pytest.mark.parametrize("softcap", [5.0, 30.0, 1000.0])
def test_logits_softcap_of_fp32_logits(D, T, softcap):
    """Small whole numbers, whose sums are exact: what is left is x / softcap (two roundings), tanh (2 steps of its
    value) and the product with the cap (half a step), at any D."""
    g = torch.Generator().manual_seed(D + T)
    e, c = (torch.randint(-2, 3, (n, D), generator=g).to(BF16) for n in (T, 300))
    x = e.double() @ c.double().T
    want = softcap * torch.tanh(x / softcap)
    got = linear_logits(e.to(DEV), c.to(DEV), softcap=softcap, out_dtype=FP32).cpu().double()
    tol = 2.5 * 2.0**-23 * want.abs() + 2.0**-23 * x.abs() * (1 - (want / softcap) ** 2)
    assert bool(((got - want).abs() <= tol * 1.01).all())


# Column widths of 16 to 256 (with an order of the adapters: up to 15 more per run), and several column tiles
WIDTHS = [10, 64, 80, 128, 144, 190, 208, 256, 300, 700]


@pytest.mark.parametrize("T", WIDTHS)
@pytest.mark.parametrize("D", [520, 1001, 1024])
@pytest.mark.parametrize("adapters", ["none", "ordered", "runs", "many", "odd_rank"])
def test_logits_fp32_of_long_reductions(T, D, adapters):
    """fp32 logits whose sums are handed over several times, with each form of the adapters' product."""
    n, r, layout = {"none": (0, 0, "each"), "ordered": (3, 24, "each"), "runs": (3, 40, "runs"),
                    "many": (200, 16, "each"), "odd_rank": (4, 12, "each")}[adapters]  # fmt: skip
    kw = _inputs(T, 700, D, FP16 if T == 128 else BF16, n=n, r=r, layout=layout, bias=FP32, seed=T + D)
    _check_logits(kw, out_dtype=FP32, softcap=20.0 if T % 3 else None)


@pytest.mark.parametrize("T", [9, 100, 150, 250])
@pytest.mark.parametrize("adapters", [0, 3])
def test_logits_fp32_of_more_tiles_than_cta_pairs(T, adapters):
    """19700 rows: 77 tiles for at most 74 pairs, 2304 reduction elements."""
    _check_logits(_inputs(T, 19_700, 2304, BF16, n=adapters, r=16, bias=BF16, seed=T), out_dtype=FP32, softcap=30.0)


@pytest.mark.parametrize("T", WIDTHS)
@pytest.mark.parametrize("D", [176, 520])
def test_logits_fp32_operands_of_long_reductions(T, D):
    """The three-term split makes 3 D of them."""
    _check_logits(_inputs(T, 600, D, FP32, n=2 if T % 2 else 0, r=8, bias=FP32, seed=T))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_logits_of_long_reductions_do_not_depend_on_the_batch_mates(dtype):
    kw = _to_dev(_inputs(700, 500, 1000, dtype))
    full = linear_logits(**kw, out_dtype=FP32)
    for n in WIDTHS:
        assert torch.equal(linear_logits(**dict(kw, e=kw["e"][:n]), out_dtype=FP32), full[:n]), n
        assert torch.equal(linear_logits(**dict(kw, e=kw["e"][700 - n :]), out_dtype=FP32), full[700 - n :]), n


@pytest.mark.parametrize("T", [5, 100, 150, 250])
@pytest.mark.parametrize("D", [256, 520, 2048])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_logits_fp32_sums_do_not_drift(T, D, dtype):
    """Whole numbers whose sums over 256 elements stay below 2^24, hence are exact on the tensor cores; the sums of these
    round to the nearest: off by at most half a step for each, and by nothing on average."""
    g = torch.Generator().manual_seed(T + D)
    e, c = (torch.randint(200, 256, (n, D), generator=g).to(dtype) for n in (T, 2000))
    parts = torch.stack([e[:, i : i + 256].double() @ c[:, i : i + 256].double().T for i in range(0, D, 256)])
    assert parts.max() < 2**24
    run = parts.cumsum(0)
    half_steps = torch.exp2(run[1:].log2().floor() - 24)  # of the results of the additions
    err = linear_logits(e.to(DEV), c.to(DEV), out_dtype=FP32).cpu().double() - run[-1]
    assert bool((err.abs() <= 1.01 * half_steps.sum(0)).all())
    # the mean of N errors bounded by b and as often up as down: 6 b / sqrt(N)
    bound = float(half_steps.sum(0).max()) if len(half_steps) else 0.0
    assert abs(float(err.mean())) <= 6 * bound / err.numel() ** 0.5


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("r", [8, 16, 48])
@pytest.mark.parametrize("exponent", [-2, -7, -8, -9, -12, -16, -20, -24, -30])
def test_logits_small_inner_products(dtype, r, exponent):
    """Adapters alone (c = 0) whose inner products h come near the end of fp16, with large entries of B.  Of h is lost, beside
    D + 2 roundings of its fp32 sum: 2^-22 or, in fp16, 2^-25 where the column's largest is 2^-8 or more; and of the second
    product a step 2^-23 for each of its up to 3 r additions."""
    T, V, D = 40, 300, 128
    kw = _inputs(T, V, D, dtype, n=2, r=r, seed=r)
    kw["c"].zero_()
    kw["adapter_ids"] = torch.arange(T) // 20
    kw["lora_b"] = (kw["lora_b"].float() * 1e4).clamp(-6e4, 6e4).to(dtype)
    kw["lora_scale"] = torch.tensor([2.0**exponent, 2.0**exponent])
    kw["lora_a"][0, 1] *= 2.0**-4  # a smaller one among the others
    ref, _ = H.linear_logits(**kw)
    A, B = (kw[k].double()[kw["adapter_ids"]] for k in ("lora_a", "lora_b"))
    e, s = kw["e"].double(), 2.0**exponent
    h = s * torch.einsum("td,trd->tr", e, A)
    h_mag = s * torch.einsum("td,trd->tr", e.abs(), A.abs())
    assert ref.abs().max() > 0
    lost = torch.full_like(h, 0.0) if dtype == BF16 else torch.where(h.abs().amax(1, keepdim=True) >= 2.0**-8 * 0.99, 2.0**-25, 0.0) + 0 * h
    h_err = (D + 2) * 2.0**-24 * h_mag + torch.maximum(2.0**-22 * h.abs(), lost)
    tol = torch.einsum("tvr,tr->tv", B.abs(), h_err + 3 * r * 2.0**-23 * h.abs())
    got = linear_logits(**_to_dev(kw), out_dtype=FP32).cpu().double()
    assert bool(((got - ref).abs() <= tol * 1.01).all())


def test_logits_output_past_two_to_the_31():
    """16384 x 140000 16-bit logits: offsets pass 2^31 elements."""
    kw = _to_dev(_inputs(16384, 140000, 64, BF16))
    got = linear_logits(**kw)
    rows = torch.tensor([0, 8191, 15338, 15339, 16383], device=DEV)
    ref, mag = H.linear_logits(kw["e"][rows].cpu(), kw["c"].cpu())
    err = (got[rows].cpu().double() - ref).abs()
    assert bool((err <= _tolerance(ref, mag, BF16, BF16, 64, None)).all())


# ---------------------------------------------------------------- sampling


def _check_sample(logits, u, **kw):
    ref_tok, ref_lp = H.sample_tokens(logits.cpu(), u.cpu(), **{k: v.cpu() if torch.is_tensor(v) else v for k, v in kw.items()})
    tok, lp = sample_tokens(logits, u, return_logprobs=True, **kw)
    assert tok.dtype == torch.int64 and lp.dtype == FP32
    assert torch.equal(tok.cpu(), ref_tok), (tok.cpu() != ref_tok).nonzero().flatten().tolist()[:8]
    lp = lp.cpu().double()
    none = torch.isinf(ref_lp)
    assert torch.equal(torch.isinf(lp), none)
    # rounding to fp32 (half a step), and weights rounded to at worst half of 2^-42 of the largest, in a sum of at least one
    tol = 2.0**-24 * ref_lp.abs() * 1.01 + 2.0**-43 * logits.size(-1) + 1e-12
    assert bool(((lp - ref_lp).abs()[~none] <= tol[~none]).all())
    assert torch.equal(sample_tokens(logits, u, **kw), tok)
    return tok


def _rows(B, V, dtype, seed=0, peak=10.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * 2.5
    x[torch.arange(B)[:, None], torch.randint(0, V, (B, min(V, 20)), generator=g)] += peak * torch.rand(B, min(V, 20), generator=g)
    return x.to(dtype).to(DEV), torch.rand(B, generator=g).to(DEV)


SETTINGS = {
    "plain": dict(),
    "cool": dict(temperature=0.3),
    "hot": dict(temperature=3.0),
    "k1": dict(top_k=1),
    "k50": dict(top_k=50),
    "k3000": dict(top_k=3000, temperature=2.0),
    "p": dict(top_p=0.9),
    "p_small": dict(top_p=0.05),
    "p_near_1": dict(top_p=0.9999, temperature=1.5),
    "min_p": dict(min_p=0.02),
    "min_p_1": dict(min_p=1.0),
    "all": dict(temperature=0.8, top_k=200, top_p=0.95, min_p=0.001),
    "greedy": dict(temperature=0.0, top_k=40, top_p=0.5),
}


@pytest.mark.parametrize("V", [1, 2, 7, 32, 511, 512, 513, 4095, 8193, 20000, 70001, 150000])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_sample_sizes(V, dtype):
    x, u = _rows(12, V, dtype, seed=V)
    for kw in SETTINGS.values():
        _check_sample(x, u, **kw)


@pytest.mark.parametrize("name", list(SETTINGS))
def test_sample_flat_and_tied(name):
    """Near-uniform rows (thousands of tokens of almost equal weight) and rows with few distinct values."""
    kw = SETTINGS[name]
    g = torch.Generator().manual_seed(3)
    u = torch.rand(16, generator=g).to(DEV)
    _check_sample((torch.randn(16, 30000, generator=g) * 0.01).to(DEV), u, **kw)
    _check_sample((torch.randn(16, 30000, generator=g) * 1e-7 + 5).to(DEV), u, **kw)
    _check_sample(torch.randint(-2, 3, (16, 30000), generator=g).float().to(DEV), u, **kw)
    _check_sample(torch.zeros(16, 30000, device=DEV), u, **kw)
    signed_zeros = torch.where(torch.rand(16, 5000, generator=g) < 0.5, -0.0, 0.0).to(DEV)
    _check_sample(signed_zeros, u, **kw)


@pytest.mark.parametrize("name", list(SETTINGS))
def test_sample_masked_and_extreme_rows(name):
    kw = SETTINGS[name]
    V = 9000
    g = torch.Generator().manual_seed(5)
    low = torch.finfo(FP32).min
    x = torch.randn(16, V, generator=g) * 3
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = low
    x[3] = -math.inf
    x[3, 8999] = -5.0
    x[4, torch.rand(V, generator=g) < 0.99] = -math.inf
    x[5, torch.rand(V, generator=g) < 0.99] = low
    x[6, torch.rand(V, generator=g) < 0.5] = math.nan
    x[7, ::1000] = math.inf
    x[8, 4321] = math.inf
    x[9] = torch.finfo(FP32).max
    x[9, ::2] = low
    x[10] *= 1e30
    x[11] *= 1e-30
    x[12] = torch.linspace(-45, 0, V)
    x[13] = 1e4 + torch.randn(V, generator=g)
    x[14] = torch.tensor([0.0, -30.0, math.nan]).repeat(V // 3)
    x[15, 1:] = -math.inf
    u = torch.rand(16, generator=g).to(DEV)
    _check_sample(x.to(DEV), u, **kw)
    tok = sample_tokens(x.to(DEV), u, **kw).cpu()
    assert tok[0] == -1 and tok[1] == -1 and tok[2] >= 0 and tok[3] == 8999 and tok[8] == 4321 and tok[15] == 0


def test_sample_border_numbers():
    x, _ = _rows(6, 5000, FP32)
    below_one = 1.0 - 2.0**-24
    for u in (0.0, below_one, 0.5, 2.0**-24):
        for kw in SETTINGS.values():
            _check_sample(x, torch.full((6,), u, device=DEV), **kw)
    # outside the documented range: the last kept token, and the first
    last = sample_tokens(x, torch.full((6,), below_one, device=DEV), top_k=3)
    for u in (1.0, 2.0, math.inf):
        assert torch.equal(sample_tokens(x, torch.full((6,), u, device=DEV), top_k=3), last)
    first = sample_tokens(x, torch.zeros(6, device=DEV), top_k=3)
    for u in (-1.0, math.nan):
        assert torch.equal(sample_tokens(x, torch.full((6,), u, device=DEV), top_k=3), first)


@pytest.mark.parametrize("T", [5e-324, 1e-310, 1e-30, 1e-3, 1e4, 1e30, 1e308, math.inf])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=77), dict(top_p=0.7), dict(top_k=999, top_p=0.3, min_p=0.5)])
def test_sample_extreme_temperatures(T, kw):
    x, u = _rows(4, 12345, FP32, seed=9)
    x[2, ::3] = -math.inf
    x[3, ::3] = torch.finfo(FP32).min
    _check_sample(x, u, temperature=T, **kw)
    _check_sample(torch.full((4, 5000), 2.5, device=DEV), u, temperature=T, **kw)  # nothing but the largest


def test_sample_every_row_has_its_own_settings():
    B, V = 64, 33333
    x, u = _rows(B, V, BF16, seed=11)
    g = torch.Generator().manual_seed(12)
    r = lambda: torch.rand(B, generator=g).to(DEV)
    kw = dict(
        temperature=torch.where(r() < 0.2, 0.0, 0.2 + 2 * r()),
        top_k=(r() ** 4 * 2 * V).long(),
        top_p=torch.where(r() < 0.3, 1.0, r()),
        min_p=torch.where(r() < 0.3, 0.0, 0.3 * r()),
    )
    tok = _check_sample(x, u, **kw)
    # a row alone gives the same token, and so do numbers in place of tensors
    for i in (0, 13, 63):
        one = {k: v[i : i + 1] for k, v in kw.items()}
        assert sample_tokens(x[i : i + 1], u[i : i + 1], **one).item() == tok[i].item()
        assert sample_tokens(x[i], u[i], **{k: v[i].item() for k, v in kw.items()}).item() == tok[i].item()
    assert torch.equal(sample_tokens(x, u, **dict(kw, top_k=kw["top_k"].int(), top_p=kw["top_p"].double())), tok)
    shaped = sample_tokens(x.view(4, 16, V), u.view(4, 16), **{k: v.view(4, 16) for k, v in kw.items()})
    assert torch.equal(shaped, tok.view(4, 16))


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_sample_strides_and_alignment(dtype):
    x, u = _rows(9, 20001, dtype, seed=2)
    kw = dict(top_k=300, top_p=0.9)
    want = sample_tokens(x, u, **kw)
    for off in range(1, 9):
        wide = torch.full((9, 20001 + 16), math.inf, dtype=dtype, device=DEV)  # must not be read as logits
        wide[:, off : off + 20001] = x
        assert torch.equal(sample_tokens(wide[:, off : off + 20001], u, **kw), want), off
    assert torch.equal(sample_tokens(x.t().contiguous().t(), u, **kw), want)
    assert torch.equal(sample_tokens(x[:1].expand(9, -1), u, **kw)[:1], want[:1])
    assert torch.equal(sample_tokens(x[::2], u[::2], **kw), want[::2])


@pytest.mark.parametrize("dtype, B", [(FP32, 70), (BF16, 140)])
@pytest.mark.parametrize("name", list(SETTINGS))
def test_sample_many_long_rows(name, dtype, B):
    """Enough logits for the streaming kernels, with odd lengths, strides and extreme rows; a row alone, which takes
    the other path, gives the same token."""
    V, kw = 120_011, SETTINGS[name]
    x, u = _rows(B, V + 3, dtype, seed=21)
    x = x[:, 1 : V + 1]
    x[0] = -math.inf
    x[1] = 2.0
    x[2] = torch.finfo(dtype).min
    x[3, ::2] = math.nan
    x[4, 5::7] = -math.inf
    x[5, 77777] = math.inf
    x[6, :] = torch.linspace(-40, 0, V, device=DEV).to(dtype)
    x[7] *= 0.001
    x[8] = torch.where(torch.arange(V, device=DEV) % 5 == 0, 1.0, -1.0).to(dtype)
    assert x.numel() * x.element_size() >= 32 << 20
    tok, lp = sample_tokens(x, u, return_logprobs=True, **kw)
    rows = list(range(12)) + list(range(12, B, 16))  # the oracle sorts in 64 bits: some of the rows
    ref_tok, ref_lp = H.sample_tokens(x[rows].cpu(), u[rows].cpu(), **kw)
    assert torch.equal(tok[rows].cpu(), ref_tok)
    finite = torch.isfinite(ref_lp)
    err = (lp[rows].cpu().double() - ref_lp).abs()[finite]
    assert bool((err <= 2.0**-24 * ref_lp.abs()[finite] * 1.01 + 2.0**-42 * V + 1e-12).all())
    for i in (0, 1, 5, 8, 30, B - 1):
        assert sample_tokens(x[i], u[i], **kw).item() == tok[i].item()


def test_sample_many_long_rows_with_their_own_settings():
    B, V = 70, 120_001
    x, u = _rows(B, V, FP32, seed=31)
    g = torch.Generator().manual_seed(32)
    r = lambda: torch.rand(B, generator=g).to(DEV)
    kw = dict(
        temperature=torch.where(r() < 0.2, 0.0, 0.2 + 2 * r()),
        top_k=torch.where(r() < 0.5, 0, (r() ** 4 * 2 * V).long()),
        top_p=torch.where(r() < 0.4, 1.0, r()),
        min_p=torch.where(r() < 0.5, 0.0, 0.3 * r()),
    )
    kw["top_k"][:5], kw["top_p"][:5] = 0, 1.0  # nothing cut off, in the company of filters
    _check_sample(x, u, **kw)


@pytest.mark.parametrize("dtype, B", [(FP32, 70), (BF16, 140)])
@pytest.mark.parametrize("min_p", [None, 0.3])
def test_sample_many_long_greedy_rows_without_filters(dtype, B, min_p):
    """Enough logits for the streaming kernels and neither top-k nor top-p: greedy rows alone and among others."""
    V = 120_011
    x, u = _rows(B, V, dtype, seed=41)
    x[0] = -math.inf
    x[1] = 2.0  # all are the largest
    x[2, [5, 60_000, 119_999]] = 90.0  # tied maxima, the first in the first chunk ..
    x[3, [119_000, 119_999]] = 90.0  # .. and both in the last one
    x[4, 1:] = -math.inf
    x[5] = math.nan
    x[5, 100_001] = -7.0
    x[6] = -0.0
    x[6, 33] = 0.0
    x[7, [77, 78]] = math.inf
    assert x.numel() * x.element_size() >= 32 << 20
    first = torch.tensor([-1, 0, 5, 119_000, 0, 100_001, 0, 77])
    tok, lp = sample_tokens(x, u, temperature=0.0, min_p=min_p, return_logprobs=True)
    assert torch.equal(tok[:8].cpu(), first)
    is_max = x[8:] == x[8:].amax(1, keepdim=True)
    assert torch.equal(tok[8:], is_max.int().argmax(1))  # the first of the largest
    assert bool((lp[1:] == 0).all()) and lp[0] == -math.inf
    for i in (0, 2, 3, 20, B - 1):
        assert sample_tokens(x[i], u[i], temperature=0.0, min_p=min_p).item() == tok[i].item()
    temperature = torch.where(torch.arange(B, device=DEV) % 3 == 1, 0.8, torch.zeros(B, device=DEV))
    temperature[3] = math.nan  # in a tensor: greedy
    mixed = sample_tokens(x, u, temperature=temperature, min_p=min_p)
    cold = ~(temperature > 0)
    assert torch.equal(mixed[cold], tok[cold])
    some = [1, 4, 7, 10, 13, 16]
    as_stored = torch.tensor(0.8).item()
    warm, _ = H.sample_tokens(x[some].cpu(), u[some].cpu(), temperature=as_stored, min_p=min_p)
    assert torch.equal(mixed[some].cpu(), warm)


@pytest.mark.parametrize("dtype, B, V", [(FP32, 300_000, 33), (BF16, 3000, 9000), (FP32, 560, 15_900), (FP16, 520, 32_500)])
@pytest.mark.parametrize("name", ["plain", "greedy", "p", "all"])
def test_sample_many_short_rows(dtype, B, V, name):
    """As many bytes as the streaming kernels begin with, in rows too short for them, or just long enough."""
    kw = SETTINGS[name]
    x, u = _rows(B, V, dtype, seed=V)
    assert x.numel() * x.element_size() >= 32 << 20
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    tok = sample_tokens(x, u, **kw)
    assert torch.cuda.max_memory_allocated() - before <= 0.6 * x.numel() * x.element_size() + 16 * B + 4096
    for lo in range(0, B, max(1, B // 5)):  # parts of the batch, too small for them
        part = slice(lo, lo + (8 << 20) // (V * x.element_size()))
        assert torch.equal(sample_tokens(x[part], u[part], **kw), tok[part])
    rows = list(range(0, B, B // 12))
    want, _ = H.sample_tokens(x[rows].cpu(), u[rows].cpu(), **kw)
    assert torch.equal(tok[rows].cpu(), want)


@pytest.mark.parametrize("name", ["plain", "greedy", "p", "all"])
def test_sample_offsets_past_two_to_the_31(name):
    """Rows more than 2^31 elements apart, and a batch of more than 2^31 logits (the streaming kernels)."""
    kw = SETTINGS[name]
    x, u = _rows(3, 20_000, BF16, seed=51)
    apart = 2**31 + 24
    far = torch.empty(apart + 40_000, dtype=BF16, device=DEV).as_strided((2, 20_000), (apart, 1))
    far.copy_(x[:2])
    assert torch.equal(sample_tokens(far, u[:2], **kw), sample_tokens(x[:2], u[:2], **kw))
    del far
    B, V = 16_400, 131_000
    few, _ = _rows(40, V, BF16, seed=52)
    big = few.repeat(B // 40, 1)
    u = torch.rand(B, generator=torch.Generator().manual_seed(53)).to(DEV)
    tok = sample_tokens(big, u, **kw)
    for rows in (slice(0, 3), slice(8000, 8003), slice(16_390, 16_400)):
        assert torch.equal(sample_tokens(few[torch.arange(B, device=DEV)[rows] % 40], u[rows], **kw), tok[rows])


def test_linear_sample_of_a_large_greedy_batch():
    """The float32 logits of 70 x 120011 go through the streaming kernels."""
    kw = _to_dev(_inputs(70, 120_011, 64, BF16))
    u = torch.rand(70, generator=torch.Generator().manual_seed(2)).to(DEV)
    x = linear_logits(**kw, out_dtype=FP32)
    tok = linear_sample(**kw, u=u, temperature=0.0)
    assert torch.equal(tok, (x == x.amax(1, keepdim=True)).int().argmax(1))  # compared, never used as an index
    assert torch.equal(tok, torch.stack([sample_tokens(x[i], u[i], temperature=0.0) for i in range(70)]))


def test_sample_empty_and_too_large():
    assert sample_tokens(torch.zeros(0, 10, device=DEV), torch.zeros(0, device=DEV)).shape == (0,)
    with pytest.raises(_native.NativeError):
        sample_tokens(torch.zeros(1, 1_000_000, device=DEV), torch.zeros(1, device=DEV))
    with pytest.raises(_native.NativeError):
        sample_tokens(torch.zeros(1, 2**20 + 1, device=DEV, dtype=BF16), torch.zeros(1, device=DEV))
    x, u = _rows(2, 2**20, BF16)
    _check_sample(x, u, top_k=20, top_p=0.9)
    x, u = _rows(2, 700_000, FP32)
    _check_sample(x, u, top_p=0.99)


def test_sample_frequencies_follow_the_weights():
    """Evenly spread numbers u give every token its share, up to one draw."""
    N = 4096
    x, _ = _rows(1, 50, FP32, seed=4, peak=2.0)
    u = (torch.arange(N, device=DEV) + 0.5) / N
    tok = sample_tokens(x.expand(N, -1).contiguous(), u.float(), temperature=2.0)
    share = torch.softmax(x[0].double() / 2, 0) * N
    assert bool(((torch.bincount(tok, minlength=50) - share).abs() <= 1.0 + 1e-6).all())


# ---------------------------------------------------------------- together


def _step_inputs(T=21, V=5003, D=320):
    kw = _inputs(T, V, D, BF16, n=3, r=16, bias=FP32)
    kw["e"] = kw["e"] * 3
    return _to_dev(kw), torch.rand(T, generator=torch.Generator().manual_seed(1)).to(DEV)


def test_linear_sample_is_the_two_operators():
    kw, u = _step_inputs()
    s = dict(temperature=0.9, top_k=100, top_p=0.95)
    tok, lp = linear_sample(**kw, u=u, softcap=30.0, return_logprobs=True, **s)
    logits = linear_logits(**kw, softcap=30.0, out_dtype=FP32)
    assert torch.equal(tok, _check_sample(logits, u, **s))
    assert torch.equal(linear_sample(**kw, u=u, softcap=30.0, **s), tok)
    assert bool((lp <= 0).all())


def test_linear_sample_on_another_stream():
    kw, u = _step_inputs()
    want = linear_sample(**kw, u=u, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_sample(**kw, u=u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_decoding_steps_captured_and_replayed():
    """Two captured steps with their own workspaces, replayed on new embeddings, adapters and numbers."""
    kw, u = _step_inputs()
    temp = torch.full((21,), 0.7, device=DEV)
    k = torch.full((21,), 40, device=DEV)
    step = lambda: linear_sample(**kw, u=u, temperature=temp, top_k=k, return_logprobs=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(step())
    g = torch.Generator().manual_seed(8)
    for i in range(4):
        kw["e"].copy_(torch.randn(21, 320, generator=g) * 3)
        kw["adapter_ids"].copy_(torch.randint(-1, 3, (21,), generator=g))
        u.copy_(torch.rand(21, generator=g))
        temp.copy_(torch.rand(21, generator=g))
        k.copy_(torch.randint(0, 100, (21,), generator=g))
        graphs[i % 2].replay()
        want = step()
        for a, b in zip(outs[i % 2], want):
            assert torch.equal(a, b)


FIRST_LAUNCH = """
import torch
from cut_cross_entropy import linear_logits, linear_sample, sample_tokens

g = torch.Generator().manual_seed(0)
r = lambda *shape: torch.randn(*shape, generator=g).to("cuda", torch.bfloat16)
e, c, a, b, u = r(250, 640), r(900, 640), r(2, 16, 640), r(2, 900, 16), torch.rand(250, generator=g).cuda()
ids = torch.arange(250, device="cuda") % 3 - 1
step = lambda: (linear_logits(e, c, lora_a=a, lora_b=b, adapter_ids=ids, out_dtype=torch.float32),
                linear_logits(e[:20], c), linear_sample(e[:70], c, u[:70], top_p=0.9), sample_tokens(r2, u[:70]))
r2 = r(70, 240_000)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
for x, y in zip(got, step()):
    assert torch.equal(x, y)
print("captured")
"""


def test_first_launch_of_every_form_inside_a_capture():
    """A process whose first calls are captured: the kernels are loaded and set up there."""
    import os
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent
    env = dict(os.environ, PYTHONPATH=str(root / "ml-cross-entropy_b200"))
    out = subprocess.run([sys.executable, "-c", FIRST_LAUNCH], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_forms_first_launched_by_two_threads_at_once():
    """Two threads on their own streams, with shapes that take different forms of the kernels."""
    import threading

    kw = _to_dev(_inputs(250, 900, 640, FP16, n=2, r=16))
    x, u = _rows(40, 9000, FP16)
    jobs = [lambda: linear_logits(**kw, out_dtype=FP32), lambda: sample_tokens(x, u, top_p=0.8),
            lambda: linear_logits(kw["e"][:100], kw["c"], out_dtype=FP32), lambda: linear_logits(**kw)]  # fmt: skip
    got: dict = {}

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [jobs[i]() for _ in range(20)]
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i, job in enumerate(jobs):
        want = job()
        assert len(got[i]) == 20 and all(torch.equal(y, want) for y in got[i])


def test_training_and_answering_share_the_head():
    """The loss's own numbers from the logits: lse and the correct-token logit agree with linear_cross_entropy."""
    from cut_cross_entropy import linear_cross_entropy

    kw = _to_dev(_inputs(64, 3001, 256, BF16, bias=FP32))
    targets = torch.randint(0, 3001, (64,), device=DEV)
    loss, lse = linear_cross_entropy(**kw, targets=targets, softcap=20.0, reduction="none", return_lse=True)
    x = linear_logits(**kw, softcap=20.0, out_dtype=FP32).double()
    # both sum 256 bf16 products in fp32: K 2^-23 of the products' magnitude each, ex2 and lg2 within 2^-20
    tol = 2 * 264 * 2.0**-23 * H.linear_logits(**{k: v.cpu() for k, v in kw.items()})[1].max().item() + 2.0**-18
    assert (torch.logsumexp(x, 1) - lse).abs().max().item() <= tol
    nll = torch.logsumexp(x, 1) - x.gather(1, targets[:, None]).squeeze(1)
    assert (nll - loss).abs().max().item() <= 2 * tol
