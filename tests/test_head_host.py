"""Head operators without a GPU: refusals, argument checks of the C entry points, the oracle's known answers."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from cut_cross_entropy import _native, linear_logits, linear_sample, sample_tokens
from cut_cross_entropy.linear_logits import _rows
from oracle import head_oracle as H


def _lora(n=2, r=8, D=16, V=10, T=4):
    return dict(lora_a=torch.zeros(n, r, D), lora_b=torch.zeros(n, V, r), adapter_ids=torch.zeros(T, dtype=torch.int64))


@pytest.mark.parametrize(
    "kw, err",
    [
        (dict(e=torch.zeros(4, 15)), ValueError),
        (dict(c=torch.zeros(10, 16, 1)), ValueError),
        (dict(bias=torch.zeros(9)), ValueError),
        (dict(softcap=0.0), ValueError),
        (dict(softcap=-1.0), ValueError),
        (dict(lora_scale=1.0), ValueError),
        (dict(_lora(), lora_b=None), ValueError),
        (dict(_lora(), adapter_ids=None), ValueError),
        (dict(_lora(r=257)), ValueError),
        (dict(_lora(n=0)), ValueError),
        (dict(_lora(D=8)), ValueError),
        (dict(_lora(V=11)), ValueError),
        (dict(_lora(T=5)), ValueError),
        (dict(_lora(), adapter_ids=torch.zeros(4)), ValueError),
        (dict(_lora(), lora_scale=torch.ones(3)), ValueError),
        (dict(e=torch.zeros(4, 16, requires_grad=True)), RuntimeError),
        (dict(), RuntimeError),  # host tensors
    ],
)
def test_linear_logits_refusals(kw, err):
    args = dict(e=torch.zeros(4, 16), c=torch.zeros(10, 16))
    args.update(kw)
    with pytest.raises(err):
        linear_logits(**args)


@pytest.mark.parametrize(
    "kw, err",
    [
        (dict(u=torch.zeros(3)), ValueError),
        (dict(u=torch.zeros(4, dtype=torch.int64)), ValueError),
        (dict(logits=torch.zeros(4, 0)), ValueError),
        (dict(temperature=-1.0), ValueError),
        (dict(temperature=math.nan), ValueError),
        (dict(top_k=-1), ValueError),
        (dict(top_k=2.5), ValueError),
        (dict(top_k=torch.ones(4)), ValueError),
        (dict(top_k=torch.ones(3, dtype=torch.int64)), ValueError),
        (dict(top_p=1.5), ValueError),
        (dict(top_p=-0.1), ValueError),
        (dict(min_p=1.1), ValueError),
        (dict(min_p=torch.ones(4, 1)), ValueError),
        (dict(temperature=torch.ones(4, dtype=torch.bool)), ValueError),
        (dict(logits=torch.zeros(4, 7, requires_grad=True)), RuntimeError),
        (dict(), RuntimeError),
    ],
)
def test_sample_tokens_refusals(kw, err):
    args = dict(logits=torch.zeros(4, 7), u=torch.zeros(4))
    args.update(kw)
    with pytest.raises(err):
        sample_tokens(**args)


@pytest.mark.parametrize("name", ["u", "temperature", "top_p", "min_p"])
def test_sample_tokens_refuses_settings_that_want_a_gradient(name):
    args = dict(logits=torch.zeros(4, 7), u=torch.zeros(4))
    args[name] = torch.full((4,), 0.5, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        sample_tokens(**args)


def test_linear_logits_refuses_a_scale_that_wants_a_gradient():
    args = dict(e=torch.zeros(4, 16), c=torch.zeros(10, 16), **_lora())
    with pytest.raises(RuntimeError, match="no backward"):
        linear_logits(**args, lora_scale=torch.ones(args["lora_a"].size(0), requires_grad=True))


@pytest.fixture(scope="module")
def as_dtensor():
    """Wraps a host tensor as a DTensor on a mesh of one rank."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import DeviceMesh
    from torch.distributed.tensor import DTensor, Replicate

    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        mesh = DeviceMesh("cpu", [0])
        yield lambda t: DTensor.from_local(t, mesh, [Replicate()])
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("name", ["e", "c", "bias", "lora_a", "lora_b", "adapter_ids", "lora_scale"])
def test_linear_logits_refuses_dtensors(name, as_dtensor):
    args = dict(e=torch.zeros(4, 16), c=torch.zeros(10, 16), bias=torch.zeros(10), **_lora(), lora_scale=torch.ones(2))
    args[name] = as_dtensor(args[name])
    with pytest.raises(ValueError, match=f"{name} as a torch.distributed.tensor.DTensor"):
        linear_logits(**args)
    with pytest.raises(ValueError, match=f"{name} as a torch.distributed.tensor.DTensor"):
        linear_sample(**args, u=torch.zeros(4))


@pytest.mark.parametrize("name", ["logits", "u", "temperature", "top_k", "top_p", "min_p"])
def test_sample_tokens_refuses_dtensors(name, as_dtensor):
    args = dict(logits=torch.zeros(4, 7), u=torch.zeros(4), temperature=torch.ones(4), top_k=torch.ones(4).long(),
                top_p=torch.ones(4), min_p=torch.zeros(4))  # fmt: skip
    args[name] = as_dtensor(args[name])
    with pytest.raises(ValueError, match=f"{name} as a torch.distributed.tensor.DTensor"):
        sample_tokens(**args)


class _Wrapper(torch.Tensor):
    """A tensor whose values are kept elsewhere."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))


class _Marked(torch.Tensor):
    """A tensor with memory of its own, of another class."""


def test_wrappers_without_memory_are_refused_and_other_subclasses_are_not():
    args = dict(e=torch.zeros(4, 16), c=torch.zeros(10, 16), bias=torch.zeros(10))
    with pytest.raises(ValueError, match="bias is a _Wrapper"):
        linear_logits(**dict(args, bias=_Wrapper(args["bias"])))
    with pytest.raises(ValueError, match="temperature is a _Wrapper"):
        sample_tokens(torch.zeros(4, 7), torch.zeros(4), temperature=_Wrapper(torch.ones(4)))
    # these get as far as host tensors do
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        linear_logits(**dict(args, bias=args["bias"].as_subclass(_Marked), c=torch.nn.Parameter(args["c"], requires_grad=False)))


@pytest.mark.parametrize("name", ["e", "c", "bias", "lora_a", "lora_b", "lora_scale"])
def test_linear_logits_refuses_tangents(name):
    import torch.autograd.forward_ad as fwd

    args = dict(e=torch.zeros(4, 16), c=torch.zeros(10, 16), bias=torch.zeros(10), **_lora(), lora_scale=torch.ones(2))
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="needs CUDA tensors"):  # no tangent in sight
            linear_logits(**args)
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        for context in (torch.enable_grad(), torch.no_grad()):
            with context, pytest.raises(RuntimeError, match="forward-mode"):
                linear_logits(**args)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: linear_logits(x, torch.zeros(10, 16)), (torch.zeros(4, 16),), (torch.ones(4, 16),))


@pytest.mark.parametrize("name", ["logits", "u", "temperature", "top_p", "min_p"])
def test_sample_tokens_refuses_tangents(name):
    import torch.autograd.forward_ad as fwd

    args = dict(logits=torch.zeros(4, 7), u=torch.zeros(4))
    with fwd.dual_level():
        args[name] = fwd.make_dual(torch.full((4, 7) if name == "logits" else (4,), 0.5), torch.ones(4, 7) if name == "logits" else torch.ones(4))
        with pytest.raises(RuntimeError, match="forward-mode"):
            sample_tokens(**args)


def test_rows_of_one_column_have_unit_stride():
    wide = torch.arange(12.0).reshape(3, 4)
    for t in (wide[:1].t(), wide.t()[:, 1:2], wide[:, 2:3], wide[:1, :1], torch.zeros(1).expand(5, 1)):
        rows = _rows(t, 1)
        assert rows.stride(1) == 1 and (rows.size(0) == 1 or rows.stride(0) >= 1)
        assert torch.equal(rows, t)


def test_linear_sample_refuses_a_u_of_another_shape():
    with pytest.raises(ValueError):
        linear_sample(torch.zeros(4, 16), torch.zeros(10, 16), torch.zeros(3))


def test_c_entry_points_check_their_arguments():
    L = _native.lib()
    bad = -1  # CCE_ERR_ARG
    assert L.cce_b200_logits(None, None, 0, None) == bad
    assert L.cce_b200_sample(None, None, 0, None) == bad
    assert L.cce_b200_sample_workspace_bytes(None) == 0
    assert L.cce_b200_logits_workspace_bytes(None) == 0

    buf = ctypes.create_string_buffer(1024)
    ptr = ctypes.addressof(buf) // 16 * 16 + 16
    aligned = (ctypes.addressof(buf) + 255) // 256 * 256  # as a workspace has to be

    def logits_args(**kw):
        a = _native.LogitsArgs()
        a.op.e = a.op.c = a.out = ptr
        a.op.n_total = a.op.n_rows = 4
        a.op.V, a.op.D, a.op.lde, a.op.ldc, a.op.dtype = 10, 16, 16, 16, _native.DT_BF16
        a.out_dtype = _native.DT_BF16
        for k, v in kw.items():
            setattr(a.op if hasattr(a.op, k) else a, k, v)
        return a

    lora = dict(lora_a=ptr, lora_b=ptr, adapter_ids=ptr, n_adapters=2, rank=8)
    assert L.cce_b200_logits_workspace_bytes(logits_args()) > 0
    # room for at least one padded fp32 row of inner products per token
    assert (L.cce_b200_logits_workspace_bytes(logits_args(n_total=1000, n_rows=1000, **lora))
            - L.cce_b200_logits_workspace_bytes(logits_args(n_total=1000, n_rows=1000))) >= 1000 * 16 * 4  # fmt: skip
    for kw in (
        dict(e=None), dict(V=0), dict(D=0), dict(lde=15), dict(n_rows=3), dict(out_dtype=3), dict(dtype=7),
        dict(lora_a=ptr), dict(lora, rank=0), dict(lora, rank=257), dict(lora, n_adapters=0),
        dict(lora, ids_dtype=2), dict(has_softcap=1, softcap=0.0),
    ):  # fmt: skip
        assert L.cce_b200_logits_workspace_bytes(logits_args(**kw)) == 0, kw
        assert L.cce_b200_logits(logits_args(**kw), ptr, 1 << 40, None) == bad, kw
    assert L.cce_b200_logits(logits_args(), None, 0, None) == bad
    assert L.cce_b200_logits(logits_args(), ptr, 0, None) == -3  # CCE_ERR_WORKSPACE
    assert L.cce_b200_logits(logits_args(n_total=0, n_rows=0), None, 0, None) == 0

    def sample_args(**kw):
        a = _native.SampleArgs()
        a.logits = a.u = a.tokens = ptr
        a.B, a.V, a.ld, a.dtype = 2, 10, 10, _native.DT_F32
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw in (dict(logits=None), dict(u=None), dict(tokens=None), dict(V=0), dict(B=-1), dict(ld=9), dict(dtype=3)):
        assert L.cce_b200_sample(sample_args(**kw), aligned, 1 << 40, None) == bad, kw
    assert L.cce_b200_sample(sample_args(logits=ptr + 2), aligned, 1 << 40, None) == -2  # CCE_ERR_ALIGN
    assert L.cce_b200_sample(sample_args(), None, 0, None) == bad
    assert L.cce_b200_sample(sample_args(), aligned, 0, None) == -3
    assert L.cce_b200_sample(sample_args(), aligned + 8, 1 << 40, None) == -2
    assert L.cce_b200_sample(sample_args(V=2**20 + 1, ld=2**21), aligned, 1 << 40, None) == -7  # CCE_ERR_TOO_LARGE
    assert L.cce_b200_sample(sample_args(B=0, logits=None), None, 0, None) == 0


@pytest.mark.parametrize("dtype, elem", [(_native.DT_F32, 4), (_native.DT_BF16, 2), (_native.DT_F16, 2)])
@pytest.mark.parametrize("B, V", [(10**6, 32), (10**7, 5), (2100, 4000), (600, 15_000), (600, 33_000), (200, 60_000), (64, 256_000), (512, 152_064), (1, 700_000)])  # fmt: skip
@pytest.mark.parametrize("filters", [dict(), dict(top_k_all=5), dict(top_p_all=0.5)])
def test_sampling_workspace_stays_below_the_logits(dtype, elem, B, V, filters):
    a = _native.SampleArgs()
    a.B, a.V, a.ld, a.dtype, a.top_p_all = B, V, V, dtype, 1.0
    for k, v in filters.items():
        setattr(a, k, v)
    got = _native.lib().cce_b200_sample_workspace_bytes(a)
    assert 0 < got <= B * V * elem // 2 + 256


def test_the_loss_does_not_depend_on_the_serving_kernels():
    """What every entry point asks of the device names none of them: they are set up at their own first launch."""
    from pathlib import Path

    src = (Path(__file__).resolve().parent.parent / "ml-cross-entropy_b200" / "csrc" / "api.cu").read_text()
    body = src[src.index("int device_info(DeviceInfo** out) {") :]
    body = body[: body.index("\n}\n")]
    assert "engine_kernel" in body
    assert "head_" not in body and "sample_" not in body


def test_struct_sizes_match_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    root = Path(__file__).resolve().parent.parent
    src = tmp_path / "s.c"
    src.write_text(
        '#include "cce_b200.h"\n#include <stdio.h>\n#include <stddef.h>\n'
        "int main(void) { printf(\"%zu %zu %zu %zu\\n\", sizeof(cce_b200_logits_args), "
        "offsetof(cce_b200_logits_args, rank), sizeof(cce_b200_sample_args), "
        "offsetof(cce_b200_sample_args, logprobs)); return 0; }\n"
    )
    subprocess.run([gcc, "-I", str(root / "include"), "-o", str(tmp_path / "s"), str(src)], check=True)
    got = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()
    A, S = _native.LogitsArgs, _native.SampleArgs
    assert [int(g) for g in got] == [ctypes.sizeof(A), A.rank.offset, ctypes.sizeof(S), S.logprobs.offset]


def test_oracle_sampling_known_answers():
    x = torch.log(torch.tensor([0.1, 0.4, 0.2, 0.3]))
    assert H.sample_row(x, 0.0)[0] == 0
    assert H.sample_row(x, 0.0999)[0] == 0 and H.sample_row(x, 0.1001)[0] == 1
    assert H.sample_row(x, 0.71)[0] == 3
    assert H.sample_row(x, 0.99, top_k=2)[0] == 3 and H.sample_row(x, 0.0, top_k=2)[0] == 1
    assert H.sample_row(x, 0.99, top_p=0.39)[0] == 1  # one token reaches it
    assert H.sample_row(x, 0.99, top_p=0.41)[0] == 3
    assert H.sample_row(x, 0.0, min_p=0.6)[0] == 1 and H.sample_row(x, 0.99, min_p=0.6)[0] == 3
    assert H.sample_row(x, 0.3, temperature=0.0) == (1, 0.0)
    assert H.sample_row(torch.full((4,), -math.inf), 0.3) == (-1, -math.inf)
    assert math.isclose(H.sample_row(x, 0.99, top_k=2)[1], math.log(0.3 / 0.7), rel_tol=1e-6)
    # equal logits: the lower index comes first
    assert H.sample_row(torch.zeros(5), 0.99, top_k=2)[0] == 1


def test_oracle_logits_known_answer():
    e = torch.tensor([[1.0, 2.0]])
    c = torch.tensor([[1.0, 0.0], [0.0, 1.0], [1.0, 1.0]])
    a, b = torch.tensor([[[1.0, 1.0]]]), torch.tensor([[[1.0], [0.0], [2.0]]])
    x, _ = H.linear_logits(e, c, bias=torch.tensor([0.5, 0.0, 0.0]), lora_a=a, lora_b=b,
                           adapter_ids=torch.tensor([0]), lora_scale=torch.tensor([2.0]))  # fmt: skip
    assert x.tolist() == [[1.0 + 0.5 + 6.0, 2.0, 3.0 + 12.0]]
