"""What the Python binding of 4-bit projections and log-probabilities checks of the tensors
it is given, before any call: no GPU. Tensors on the CPU stand in for tensors on the GPU, and
a recorder for the library's entry points."""
import types

import numpy as np
import pytest
import torch

import hy3_amd as H

U8, I16, I32, BF16, F16 = torch.uint8, torch.int16, torch.int32, torch.bfloat16, torch.float16


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
    monkeypatch.setattr(H, "_lib", types.SimpleNamespace(
        hy3x_linear4_set=record, hy3x_logprobs=record,
        hy3x_logprobs_workspace=lambda T, V, top: 64 if 0 < T < 9 else 0))
    return seen


@pytest.fixture
def handle(calls):
    h = H.Linear4.__new__(H.Linear4)
    h._h, h.d_out, h.d_in, h.group, h.dtype = None, 96, 65, 32, "bf16"
    h._apply = lambda *args: calls.append(args) or 0
    return h


# ---------------------------------------------------------------- weights
def test_set_on_the_device(calls, handle):
    q, s, z = on_gpu(96, 33, dtype=U8), on_gpu(96, 3, dtype=BF16), on_gpu(96, 3, dtype=U8)
    handle.set(q, s, z, on_device=True)
    handle.set(q, s, on_device=True)
    handle.set(on_gpu(96 * 33, dtype=U8), s, on_device=True)
    handle.set(4096, 8192, on_device=True)
    assert calls == [(None, q.data_ptr(), s.data_ptr(), z.data_ptr(), 1),
                     (None, q.data_ptr(), s.data_ptr(), None, 1),
                     (None, calls[2][1], s.data_ptr(), None, 1), (None, 4096, 8192, None, 1)]
    good = dict(q=q, scales=s, zeros=z)
    for bad in (dict(q=torch.zeros(96, 33, dtype=U8)), dict(q=on_gpu(96, 33)),
                dict(scales=on_gpu(96, 3, dtype=F16)), dict(scales=on_gpu(96, 3, dtype=I16)),
                dict(scales=torch.zeros(96, 3, dtype=BF16)), dict(zeros=on_gpu(96, 3)),
                dict(zeros=torch.zeros(96, 3, dtype=U8))):
        with pytest.raises(TypeError):
            handle.set(**{**good, **bad}, on_device=True)
    for bad in (dict(q=on_gpu(96, 32, dtype=U8)), dict(q=on_gpu(33, 96, dtype=U8)),
                dict(q=OnGPU(torch.zeros(96, 40, dtype=U8)[:, :33])),
                dict(scales=on_gpu(96, 2, dtype=BF16)), dict(zeros=on_gpu(96, 4, dtype=U8)),
                dict(zeros=OnGPU(torch.zeros(96, 6, dtype=U8)[:, ::2]))):
        with pytest.raises(ValueError):
            handle.set(**{**good, **bad}, on_device=True)
    assert len(calls) == 4


def test_set_from_arrays(calls, handle):
    q, s, z = (np.zeros((96, n), t) for n, t in ((33, np.uint8), (3, np.int16), (3, np.uint8)))
    handle.set(q, s, z)
    handle.set(q, s.view(np.uint16))
    assert calls[0] == (None, q.ctypes.data, s.ctypes.data, z.ctypes.data, 0)
    assert calls[1][3] is None
    for bad in (dict(q=q.astype(np.int16)), dict(scales=s.astype(np.float32)),
                dict(scales=s.astype(np.float16)), dict(zeros=z.astype(np.float32)), dict(q=4096)):
        with pytest.raises(TypeError):
            handle.set(**{**dict(q=q, scales=s, zeros=z), **bad})
    for bad in (dict(q=q[:, :32]), dict(q=q[:95]), dict(scales=s[:, :2]), dict(zeros=z[:1])):
        with pytest.raises(ValueError):
            handle.set(**{**dict(q=q, scales=s, zeros=z), **bad})
    assert len(calls) == 2


# ---------------------------------------------------------------- their product
def apply_args(**change):
    return dict(dict(x=on_gpu(5, 65, dtype=BF16), y=on_gpu(5, 96), T=5), **change)


@pytest.mark.parametrize("named", [{}, dict(x_dtype="bf16"), dict(y_dtype="f32")])
def test_apply_types(calls, handle, named):
    handle.apply(**apply_args(base=on_gpu(5, 96)), **named)
    assert (calls[0][2], calls[0][7]) == (H.DTYPES["bf16"], H.DTYPES["f32"])
    for bad in (dict(x=torch.zeros(5, 65, dtype=BF16)), dict(x=on_gpu(5, 65, dtype=U8)),
                dict(x=np.zeros((5, 65), np.float32)), dict(y=torch.zeros(5, 96)),
                dict(y=on_gpu(5, 96, dtype=torch.float64)), dict(y=np.zeros((5, 96), np.float32)),
                dict(base=torch.zeros(5, 96)), dict(base=on_gpu(5, 96, dtype=BF16)),
                dict(base=np.zeros((5, 96), np.float32))):
        with pytest.raises(TypeError):
            handle.apply(**apply_args(**bad), **named)
    for kind, other in (("x_dtype", "f32"), ("y_dtype", "f16")):
        with pytest.raises(TypeError):
            handle.apply(**apply_args(), **{kind: other})
    assert len(calls) == 1


def test_apply_takes_the_rows_as_they_lie(calls, handle):
    x = OnGPU(torch.zeros(5, 100, dtype=F16)[:, 7:72])
    y, base = OnGPU(torch.zeros(5, 300)[:, :96]), OnGPU(torch.zeros(5, 200)[:, 3:99])
    handle.apply(x, y, 5, base=base, stream=77)
    assert calls[0] == (None, x.data_ptr(), H.DTYPES["f16"], 100, base.data_ptr(), 200,
                        y.data_ptr(), H.DTYPES["f32"], 300, 5, 77)
    handle.apply(x, y, 2, base=y, y_stride=300, base_stride=300)
    handle.apply(4096, 8192, 5, base=16384)
    handle.apply(4096, 8192, 5, x_dtype="f32", x_stride=70)
    assert calls[1][4:6] == (y.data_ptr(), 300) and calls[1][8] == 300
    assert calls[2][1:9] == (4096, H.DTYPES["bf16"], 65, 16384, 96, 8192, H.DTYPES["bf16"], 96)
    assert calls[3][2:4] == (H.DTYPES["f32"], 70) and calls[3][4] is None


@pytest.mark.parametrize("named", [{}, dict(x_dtype="bf16", y_dtype="f32")])
def test_apply_refuses_rows_that_are_not_there(calls, handle, named):
    for bad in (dict(T=6), dict(x=on_gpu(4, 65, dtype=BF16)), dict(x=on_gpu(5, 66, dtype=BF16)),
                dict(x=OnGPU(torch.zeros(65, 5, dtype=BF16).t())), dict(x_stride=66),
                dict(y=on_gpu(5, 95)), dict(y=on_gpu(4, 96)), dict(y_stride=97),
                dict(base=on_gpu(1, 96)), dict(base=on_gpu(5, 97)),
                dict(base=on_gpu(5, 96), base_stride=98)):
        with pytest.raises(ValueError):
            handle.apply(**apply_args(**bad), **named)
    assert not calls


def test_a_closed_projection_is_refused():
    h = H.Linear4.__new__(H.Linear4)
    h._h, h.d_out, h.d_in, h.group, h.dtype = None, 96, 65, 32, "bf16"
    h._apply = H.lib().hy3x_linear4_apply
    with pytest.raises(H.HY3XError, match="NULL"):
        h.apply(4096, 8192, 1)
    with pytest.raises(H.HY3XError, match="NULL"):
        h.set(4096, 8192, on_device=True)
    h.close()


# ---------------------------------------------------------------- log-probabilities
def row_args(**change):
    return dict(dict(logits=on_gpu(5, 70), tokens=on_gpu(5, dtype=I32), T=5, logp=on_gpu(5),
                     workspace=on_gpu(64, dtype=U8)), **change)


def alternatives(n):
    return dict(top_ids=on_gpu(5, n, dtype=I32), top_logp=on_gpu(5, n))


def test_logprobs_arguments(calls):
    a = row_args(entropy=on_gpu(5), **alternatives(4))
    H.logprobs(**a, stream=9)
    assert calls[0] == (a["logits"].data_ptr(), H.DTYPES["f32"], 70, 70, a["tokens"].data_ptr(), 5,
                        4, a["logp"].data_ptr(), a["entropy"].data_ptr(), a["top_ids"].data_ptr(),
                        a["top_logp"].data_ptr(), a["workspace"].data_ptr(), 64, 9)
    wide = OnGPU(torch.zeros(5, 90, dtype=F16)[:, 3:73])
    H.logprobs(**row_args(logits=wide, workspace=None))
    assert calls[1][:4] == (wide.data_ptr(), H.DTYPES["f16"], 90, 70)
    assert calls[1][6] == 0 and calls[1][8:13] == (None, None, None, None, 0)
    H.logprobs(4096, 8192, 5, 12288, vocab=70, top=2, top_ids=16384, top_logp=20480,
               workspace=32768, dtype="bf16", row_stride=72)
    assert calls[2] == (4096, H.DTYPES["bf16"], 72, 70, 8192, 5, 2, 12288, None, 16384, 20480,
                        32768, 64, None)
    H.logprobs(**row_args(**alternatives(6)), top=3)  # room for more
    assert calls[3][6] == 3


def test_logprobs_types(calls):
    for bad in (dict(logits=torch.zeros(5, 70)), dict(logits=on_gpu(5, 70, dtype=I32)),
                dict(logits=np.zeros((5, 70), np.float32)), dict(tokens=on_gpu(5, dtype=torch.int64)),
                dict(tokens=torch.zeros(5, dtype=I32)), dict(logp=on_gpu(5, dtype=F16)),
                dict(logp=torch.zeros(5)), dict(entropy=on_gpu(5, dtype=BF16)),
                dict(top_ids=on_gpu(5, 2), top_logp=on_gpu(5, 2)),
                dict(top_ids=on_gpu(5, 2, dtype=I32), top_logp=on_gpu(5, 2, dtype=F16)),
                dict(workspace=on_gpu(64)), dict(workspace=torch.zeros(64, dtype=U8))):
        with pytest.raises(TypeError):
            H.logprobs(**row_args(**bad))
    with pytest.raises(TypeError):
        H.logprobs(**row_args(), dtype="bf16")
    assert not calls


def test_logprobs_sizes(calls):
    for bad in (dict(T=6), dict(logits=on_gpu(4, 70)), dict(logits=OnGPU(torch.zeros(70, 5).t())),
                dict(vocab=71), dict(row_stride=71), dict(tokens=on_gpu(4, dtype=I32)),
                dict(tokens=OnGPU(torch.zeros(10, dtype=I32)[::2])), dict(logp=on_gpu(4)),
                dict(entropy=on_gpu(4)), dict(top_ids=on_gpu(5, 2, dtype=I32)),
                dict(top_logp=on_gpu(5, 2)), dict(top=2),
                dict(top_ids=on_gpu(4, 2, dtype=I32), top_logp=on_gpu(5, 2)),
                dict(top_ids=on_gpu(5, 2, dtype=I32), top_logp=on_gpu(4, 2)),
                dict(top_ids=on_gpu(5, 0, dtype=I32), top_logp=on_gpu(5, 0)),
                dict(logits=4096), dict(top_ids=4096, top_logp=8192),
                dict(workspace=OnGPU(torch.zeros(128, dtype=U8)[::2]))):
        with pytest.raises(ValueError):
            H.logprobs(**row_args(**bad))
    assert not calls
