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


# ---------------------------------------------------------------- strides and sizes
def part(rows, wide, cols, at=0, dtype=torch.float32):
    """Columns of a wider buffer."""
    return OnGPU(torch.zeros(rows, wide, dtype=dtype)[:, at:at + cols])


def test_route_takes_the_rows_as_they_lie(calls):
    wide, one = part(5, 256, 192, 3), part(1, 256, 192)
    H.route_experts(SPEC, **route_args(logits=wide))
    H.route_experts(SPEC, **route_args(logits=wide, row_stride=256))
    H.route_experts(SPEC, **route_args(logits=wide, T=2))
    H.route_experts(SPEC, **route_args(logits=one, T=1))
    H.route_experts(SPEC, **route_args(logits=on_gpu(5 * 192)))          # dense, flat
    H.route_experts(SPEC, **route_args(logits=on_gpu(5, 1, 192)))        # dense, more axes
    H.route_experts(SPEC, **route_args(logits=on_gpu(5, 256), row_stride=256))
    H.route_experts(SPEC, **route_args(logits=part(1, 5 * 256, 192), row_stride=256))
    H.route_experts(SPEC, **route_args(logits=on_gpu(5, 192), T=0))
    assert [c[3] for c in calls] == [256, 256, 256, 192, 192, 192, 256, 256, 192]
    assert calls[0][1] == wide.data_ptr()
    # one row for all tokens: its stride of 0 reaches the library, which refuses it
    for named in ({}, dict(row_stride=0), dict(dtype="f32"), dict(dtype="f32", row_stride=0)):
        H.route_experts(SPEC, **route_args(logits=OnGPU(torch.zeros(1, 192).expand(5, 192))), **named)
        assert calls[-1][3] == 0
    # one expert: a column of anything
    H.route_experts(H.RouteSpec(1, 1), OnGPU(torch.zeros(5, 3)[:, 1:2]),
                    5, on_gpu(5, dtype=I32), on_gpu(5))
    assert calls[-1][3] == 3


@pytest.mark.parametrize("named", [{}, dict(dtype="f32")])
def test_route_refuses_rows_that_are_not_there(calls, named):
    for bad in (dict(logits=on_gpu(4, 192)), dict(logits=on_gpu(5, 256)), dict(logits=on_gpu(5, 96)),
                dict(logits=OnGPU(torch.zeros(192, 5).t())), dict(logits=part(5, 256, 191)),
                dict(logits=part(4, 256, 192)), dict(logits=OnGPU(torch.zeros(5, 384)[:, ::2])),
                dict(logits=OnGPU(torch.zeros(5, 384)[:, ::2]), row_stride=384),
                dict(logits=on_gpu(5, 192), row_stride=193), dict(logits=on_gpu(5 * 192 - 1)),
                dict(logits=part(5, 256, 192, 64), row_stride=257),
                dict(logits=OnGPU(torch.zeros(5, 2, 400)[:, :, :192])),
                dict(ids=on_gpu(5, 7, dtype=I32)), dict(ids=part(5, 16, 8, dtype=I32)),
                dict(ids=on_gpu(4, 8, dtype=I32)), dict(w=on_gpu(39)), dict(w=part(5, 9, 8)),
                dict(bias=on_gpu(191)), dict(bias=OnGPU(torch.zeros(384)[::2])), dict(T=6)):
        with pytest.raises(ValueError):
            H.route_experts(SPEC, **route_args(**bad), **named)
    assert not calls


def test_apply_takes_the_rows_as_they_lie(calls, handle):
    x, base = part(5, 100, 64, 7, BF16), part(5, 200, 96, 0, BF16)
    y = part(5, 300, 96, 5, BF16)
    handle.apply(**apply_args(x=x, base=base, y=y))
    handle.apply(**apply_args(x=x, base=y, y=y, x_stride=100, y_stride=300))
    handle.apply(**apply_args(ids=on_gpu(9, dtype=I32)))
    assert [(c[4], c[9]) for c in calls] == [(100, 300), (100, 300), (64, 96)]
    assert [c[6] for c in calls[:2]] == [200, 300] and calls[2][5] is None
    assert (calls[0][2], calls[0][5], calls[0][7]) == (x.data_ptr(), base.data_ptr(), y.data_ptr())
    handle.apply(4096, 8192, 16384, 5, base=32768)
    assert (calls[-1][4], calls[-1][6], calls[-1][9]) == (64, 96, 96)


@pytest.mark.parametrize("named", [{}, dict(x_dtype="bf16", y_dtype="bf16")])
def test_apply_refuses_rows_that_are_not_there(calls, handle, named):
    for bad in (dict(ids=on_gpu(4, dtype=I32)), dict(ids=OnGPU(torch.zeros(10, dtype=I32)[::2])),
                dict(x=on_gpu(4, 64, dtype=BF16)), dict(x=on_gpu(5, 65, dtype=BF16)),
                dict(x=OnGPU(torch.zeros(64, 5, dtype=BF16).t())), dict(x=part(4, 100, 64, dtype=BF16)),
                dict(x_stride=65), dict(y=on_gpu(5, 95, dtype=BF16)), dict(y_stride=97),
                dict(y=part(5, 100, 95, dtype=BF16)), dict(base=on_gpu(4, 96, dtype=BF16)),
                dict(base=on_gpu(5, 97, dtype=BF16)), dict(base=on_gpu(5, 96, dtype=BF16), base_stride=98),
                dict(base=on_gpu(1, 96, dtype=BF16)), dict(T=6)):
        with pytest.raises(ValueError):
            handle.apply(**apply_args(**bad), **named)
    assert not calls


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7])
def test_parts_of_wider_buffers_on_the_gpu(T):
    assert torch.cuda.is_available(), "no GPU"
    g = torch.Generator().manual_seed(T)
    wide = torch.randn(T, 256, generator=g).cuda()
    got, want = ([torch.zeros(T, 8, dtype=I32, device="cuda"), torch.zeros(T, 8, device="cuda")]
                 for _ in range(2))
    H.route_experts(SPEC, wide[:, 20:212], T, *got)
    H.route_experts(SPEC, wide[:, 20:212].contiguous(), T, *want)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    h = H.Adapters(2, 8, 64, 96)
    for i in range(2):
        h.set(i, torch.randn(8, 64, generator=g).bfloat16().cuda(),
              torch.randn(96, 8, generator=g).bfloat16().cuda(), on_device=True)
    x = torch.randn(T, 80, generator=g).bfloat16().cuda()[:, 3:67]
    base = torch.randn(T, 100, generator=g).bfloat16().cuda()[:, 1:97]
    y = torch.full((T, 120), 5.0, dtype=BF16, device="cuda")
    ids = (torch.arange(T) % 3 - 1).int().cuda()
    dense = torch.zeros(T, 96, dtype=BF16, device="cuda")
    h.apply(ids, x, y[:, 7:103], T, base=base)
    h.apply(ids, x.contiguous(), dense, T, base=base.contiguous())
    torch.cuda.synchronize()
    assert torch.equal(y[:, 7:103], dense)
    assert (y[:, :7] == 5.0).all() and (y[:, 103:] == 5.0).all()
    h.close()


# ---------------------------------------------------------------- the layer's adapters
@pytest.fixture
def layer(calls, monkeypatch):
    L = H.MoELayer.__new__(H.MoELayer)
    L._h = None

    def record(*args):
        calls.append(args)
        return 0
    for name in ("forward", "forward_static", "forward_residual", "forward_adapters",
                 "set_adapters", "time_stage"):
        setattr(H._lib, "hy3x_layer_" + name, record)
    setattr(H._lib, "hy3x_layers_time_stage", record)
    return L


def test_layer_adapter_ids(calls, layer):
    ids = on_gpu(6, dtype=I32)
    layer.forward_adapters(4096, ids, 5)
    layer.forward_adapters(4096, 8192, 5)
    assert [c[3] for c in calls] == [ids.data_ptr(), 8192]
    for bad in (torch.zeros(5, dtype=I32), on_gpu(5, dtype=torch.int64), on_gpu(5),
                np.zeros(5, np.int32)):
        with pytest.raises(TypeError):
            layer.forward_adapters(4096, bad, 5)
    for bad in (on_gpu(4, dtype=I32), OnGPU(torch.zeros(10, dtype=I32)[::2])):
        with pytest.raises(ValueError):
            layer.forward_adapters(4096, bad, 5)
    assert len(calls) == 2


def open_handle():
    h = H.Adapters.__new__(H.Adapters)
    h._h = 4096
    return h


def closed(h):
    h._h = None  # as close() leaves it


def test_closed_adapters_of_a_layer(calls, layer):
    """Closed after they were set: refused by every call that would launch them."""
    gate, down = open_handle(), open_handle()
    try:
        layer.set_adapters("gate", gate)
        layer.set_adapters("down", down)
        layer.forward_adapters(4096, 8192, 5)
        layer.time_stage("gateup", 1)
        closed(gate)
        n = len(calls)
        for call in (lambda: layer.forward_adapters(4096, 8192, 5),
                     lambda: layer.time_stage("gateup", 1),
                     lambda: H.layers_time_stage([layer], "gateup", 1)):
            with pytest.raises(H.HY3XError, match="closed"):
                call()
        layer.set_adapters("gate", None)  # the last forward's replay still has it
        with pytest.raises(H.HY3XError, match="closed"):
            layer.time_stage("combine", 1)
        assert len(calls) == n + 1
        layer.forward_adapters(4096, 8192, 5)
        layer.time_stage("gateup", 1)
        for run in (lambda: layer.forward(4096, 5), lambda: layer.forward_static(4096, 5),
                    lambda: layer.forward_residual(4096, 8192, 5)):
            closed(down)
            with pytest.raises(H.HY3XError, match="closed"):
                layer.forward_adapters(4096, 16384, 5)
            run()  # uses no adapters, and nor does its replay
            layer.time_stage("gateup", 1)
            down._h = 4096
    finally:
        closed(gate), closed(down)


def test_a_layer_keeps_the_adapters_of_its_last_forward(layer):
    import gc
    import weakref
    h = open_handle()
    alive = weakref.ref(h)
    h.close = lambda: None
    layer.set_adapters("up", h)
    layer.forward_adapters(4096, 8192, 5)
    layer.set_adapters("up", None)
    del h
    gc.collect()
    assert alive() is not None  # its replay launches them
    closed(alive())
    layer.forward(4096, 5)
    gc.collect()
    assert alive() is None


# ---------------------------------------------------------------- weights
def test_set_takes_weights_of_its_own_type_and_shape(calls, handle):
    a, b = np.zeros((8, 64), np.uint16), np.zeros((96, 8), np.int16)
    handle.set(1, a, b)
    handle.set(1, a.ravel(), b.ravel())
    handle.set(1, a[None], b[:, None])
    handle.set(1, on_gpu(8, 64, dtype=BF16), on_gpu(96, 8, dtype=BF16), on_device=True)
    handle.set(1, 4096, 8192, on_device=True)
    assert calls[-1][2:4] == (4096, 8192) and len(calls) == 5
    for bad in ((a.astype(np.float16), b), (a, b.astype(np.float16)), (a.astype(np.float32), b),
                (a.astype(np.uint8), b)):
        with pytest.raises(TypeError):
            handle.set(1, *bad)
    for bad in ((a.T, b), (a, b.T), (a[:7], b), (a, b[:95]), (a.reshape(4, 128), b),
                (a[:, :32].astype(np.uint32), b)):
        with pytest.raises(ValueError):
            handle.set(1, *bad)
    ad, bd = torch.zeros(8, 64, dtype=BF16), torch.zeros(96, 8, dtype=BF16)
    for bad in ((OnGPU(ad.t().contiguous()), OnGPU(bd)), (OnGPU(ad), OnGPU(bd.t().contiguous())),
                (OnGPU(torch.zeros(64, 8, dtype=BF16).t()), OnGPU(bd)), (OnGPU(ad[:7]), OnGPU(bd))):
        with pytest.raises(ValueError):
            handle.set(1, *bad, on_device=True)
    handle.dtype = "f16"
    handle.set(1, a.astype(np.float16), b)
    assert len(calls) == 6


def test_pointers_of_what_the_binding_takes(calls):
    H.route_experts(SPEC, **route_args())  # has met fp32 and int32 tensors
    for t in (torch.zeros(3), torch.zeros(3, dtype=I32), torch.zeros(3, dtype=torch.uint8)):
        assert H._ptr(t) == H._dev(t) == t.data_ptr()
    n = np.zeros(3, np.float32)
    assert H._ptr(n) == n.ctypes.data and H._ptr(np.int64(4096)) == H._dev(np.int64(4096)) == 4096
    assert H._ptr(None) is H._dev(None) is None and H._ptr(4096) == H._dev(4096) == 4096


# ---------------------------------------------------------------- devices
class OnOther(OnGPU):
    device = "cuda:1"

    def get_device(self):
        return 1


@pytest.mark.parametrize("named", [False, True])
def test_tensors_of_another_device(calls, handle, layer, monkeypatch, named):
    """Refused unless their device is the current one, where the kernels run."""
    monkeypatch.setattr(H, "_gpus", 2)
    now = [0]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    kinds = dict(dtype="f32") if named else {}
    types = dict(x_dtype="bf16", y_dtype="bf16") if named else {}
    route = route_args(bias=on_gpu(192))
    apply = apply_args(base=on_gpu(5, 96, dtype=BF16))
    H.route_experts(SPEC, **route, **kinds)
    handle.apply(**apply, **types)
    for name in ("logits", "ids", "w", "bias"):
        with pytest.raises(ValueError, match="current device"):
            H.route_experts(SPEC, **dict(route, **{name: OnOther(route[name].t)}), **kinds)
    for name in ("ids", "x", "y", "base"):
        with pytest.raises(ValueError, match="current device"):
            handle.apply(**dict(apply, **{name: OnOther(apply[name].t)}), **types)
    a, b = torch.zeros(8, 64, dtype=BF16), torch.zeros(96, 8, dtype=BF16)
    with pytest.raises(ValueError, match="current device"):
        handle.set(0, OnGPU(a), OnOther(b), on_device=True)
    with pytest.raises(ValueError, match="current device"):
        layer.forward_adapters(4096, OnOther(apply["ids"].t), 5)
    assert len(calls) == 2
    now[0] = 1
    H.route_experts(SPEC, **{k: OnOther(v.t) if k != "T" else v for k, v in route.items()}, **kinds)
    with pytest.raises(ValueError, match="current device"):
        H.route_experts(SPEC, **route, **kinds)
    assert len(calls) == 3
