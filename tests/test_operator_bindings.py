"""What the Python binding of the operators checks of the tensors it is given, before
any call: no GPU. Tensors on the CPU stand in for tensors on the GPU, and a recorder
for the library's entry points."""
import types

import numpy as np
import pytest
import torch

import hy3_amd as H


class OnGPU:
    """A CPU tensor that says it lives on the GPU."""

    is_cuda, device = True, "cuda:0"

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return 0


def on_gpu(*shape, dtype=torch.float32):
    return OnGPU(torch.zeros(*shape, dtype=dtype))


@pytest.fixture
def calls(monkeypatch):
    """The arguments of the calls that reach the library."""
    seen = []

    def record(*args):
        seen.append(args)
        return 0
    monkeypatch.setattr(H, "_lib", types.SimpleNamespace(hy3x_route_experts=record,
                                                         hy3x_adapters_set=record))
    return seen


@pytest.fixture
def handle(calls):
    h = H.Adapters.__new__(H.Adapters)
    h._h, h.count, h.rank, h.d_in, h.d_out, h.dtype = None, 4, 8, 64, 96, "bf16"
    h._apply = lambda *args: calls.append(args) or 0
    return h


SPEC = H.RouteSpec(192, 8)
I32, BF16 = torch.int32, torch.bfloat16


def route_args(**change):
    return dict(dict(logits=on_gpu(5, 192), T=5, ids=on_gpu(5, 8, dtype=I32), w=on_gpu(5, 8)),
                **change)


def apply_args(**change):
    return dict(dict(ids=on_gpu(5, dtype=I32), x=on_gpu(5, 64, dtype=BF16),
                     y=on_gpu(5, 96, dtype=BF16), T=5), **change)


# ---------------------------------------------------------------- types and places
@pytest.mark.parametrize("named", [{}, dict(dtype="f32")])
def test_route_types(calls, named):
    H.route_experts(SPEC, **route_args(bias=on_gpu(192)), **named)
    assert len(calls) == 1 and calls[0][2] == H.DTYPES["f32"]
    for bad in (dict(logits=torch.zeros(5, 192)), dict(logits=on_gpu(5, 192, dtype=torch.int32)),
                dict(logits=on_gpu(5, 192, dtype=torch.float64)),
                dict(ids=torch.zeros(5, 8, dtype=I32)), dict(ids=on_gpu(5, 8, dtype=torch.int64)),
                dict(w=torch.zeros(5, 8)), dict(w=on_gpu(5, 8, dtype=torch.float64)),
                dict(bias=torch.zeros(192)), dict(bias=on_gpu(192, dtype=torch.float64)),
                dict(logits=np.zeros((5, 192), np.float32)), dict(ids=np.zeros((5, 8), np.int32)),
                dict(w=np.zeros((5, 8), np.float32)), dict(bias=np.zeros(192, np.float32))):
        with pytest.raises(TypeError):
            H.route_experts(SPEC, **route_args(**bad), **named)
    with pytest.raises(TypeError, match="logits"):
        H.route_experts(SPEC, **route_args(), dtype="bf16")
    assert len(calls) == 1


@pytest.mark.parametrize("named", [{}, dict(x_dtype="bf16"), dict(y_dtype="bf16"),
                                   dict(x_dtype="bf16", y_dtype="bf16")])
def test_apply_types(calls, handle, named):
    handle.apply(**apply_args(base=on_gpu(5, 96, dtype=BF16)), **named)
    assert len(calls) == 1
    for bad in (dict(ids=torch.zeros(5, dtype=I32)), dict(ids=on_gpu(5, dtype=torch.int64)),
                dict(ids=np.zeros(5, np.int32)), dict(x=torch.zeros(5, 64, dtype=BF16)),
                dict(x=on_gpu(5, 64, dtype=torch.float64)), dict(x=np.zeros((5, 64), np.float32)),
                dict(y=torch.zeros(5, 96, dtype=BF16)), dict(y=on_gpu(5, 96, dtype=torch.int16)),
                dict(y=np.zeros((5, 96), np.float32)), dict(base=torch.zeros(5, 96, dtype=BF16)),
                dict(base=on_gpu(5, 96)), dict(base=np.zeros((5, 96), np.float32))):
        with pytest.raises(TypeError):
            handle.apply(**apply_args(**bad), **named)
    for kind in ("x_dtype", "y_dtype"):
        with pytest.raises(TypeError):
            handle.apply(**apply_args(), **{kind: "f32"})
    assert len(calls) == 1


def test_pointers_have_the_named_or_the_default_type(calls, handle):
    H.route_experts(SPEC, 4096, 5, 8192, 16384, bias=32768)
    H.route_experts(SPEC, 4096, 5, 8192, 16384, dtype="f16")
    assert [c[2] for c in calls] == [H.DTYPES["f32"], H.DTYPES["f16"]]
    assert calls[0][1::2] == (4096, 192, 5, 16384) and calls[0][4] == 32768
    handle.apply(4096, 8192, 16384, 5)
    handle.apply(4096, 8192, 16384, 5, x_dtype="f32", base=32768)
    assert [c[3] for c in calls[2:]] == [H.DTYPES["bf16"], H.DTYPES["f32"]]
    assert [c[8] for c in calls[2:]] == [H.DTYPES["bf16"]] * 2
