"""hy3x_adapters_* against y = base + scale_a B_a (A_a x) in 64 bits.

The tolerance of an element counts fp32 roundings (2^-24 each, half a step) on
the absolute values that meet in it, S = |scale| sum |B| (sum |A| |x|): chains of
d_in / 32 sums and a few joins for u, `rank` sums and a few more for B u; the
base's sum rounds base + delta, and y's type its own half step."""
import ctypes

import numpy as np
import pytest

import hy3_amd as H

HALF = 2.0 ** -24


def test_create_refusals():
    lib, h = H.lib(), ctypes.c_void_p(1)
    for args, word in [((0, 8, 64, 64, 2), b"count"), ((65537, 8, 64, 64, 2), b"count"),
                       ((1, 0, 64, 64, 2), b"rank"), ((1, 129, 64, 64, 2), b"rank"),
                       ((1, 8, 0, 64, 2), b"d_in"), ((1, 8, 64, 65537, 2), b"d_out"),
                       ((1, 8, 64, 64, 0), b"type"), ((1, 8, 64, 64, 3), b"type")]:
        assert lib.hy3x_adapters_create(ctypes.byref(h), *args) == -1
        assert word in lib.hy3x_last_error() and not h.value
    assert lib.hy3x_adapters_create(None, 1, 8, 64, 64, 2) == -1


def test_null_refusals():
    lib = H.lib()
    assert lib.hy3x_adapters_destroy(None) == 0
    assert lib.hy3x_adapters_set(None, 0, None, None, 1.0, 0) == -1
    assert lib.hy3x_adapters_apply(None, 4096, 4096, 0, 64, None, 64, 8192, 0, 64, 1, None) == -1


def test_host_memory_refusals():
    import torch
    h = H.Adapters.__new__(H.Adapters)  # no GPU, no handle: refused before it is used
    h._h, h.rank, h.d_in, h.d_out, h.dtype = None, 8, 64, 96, "bf16"
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    ids = torch.zeros(1, dtype=torch.int32)
    for args in ((ids, 4096, 8192), (4096, x, 8192), (4096, 8192, x),
                 (ids.numpy(), 4096, 8192), (4096, np.zeros(64, np.float32), 8192)):
        h._apply = None
        with pytest.raises(TypeError):
            h.apply(*args, 1)
    with pytest.raises(TypeError):
        h.apply(4096, 8192, 16384, 1, base=x)
    with pytest.raises(TypeError):
        h.set(0, np.zeros((8, 64), np.uint16), np.zeros((96, 8), np.uint16), on_device=True)
    with pytest.raises(TypeError):
        h.set(0, torch.zeros(8, 64, dtype=torch.bfloat16), 4096, on_device=True)


# ---------------------------------------------------------------- on the GPU
@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


def dtype_of(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Setup:
    """A handle with random adapters, and its tensors in 64 bits on the host."""

    def __init__(self, torch, count, rank, d_in, d_out, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        t = dtype_of(torch, dtype)
        self.torch, self.dtype, self.g = torch, dtype, g
        self.a = (torch.randn(count, rank, d_in, generator=g) / d_in ** 0.5).to(t)
        self.b = (torch.randn(count, d_out, rank, generator=g) / rank ** 0.5).to(t)
        self.scale = [0.5 * (i + 1) for i in range(count)]
        self.h = H.Adapters(count, rank, d_in, d_out, dtype)
        for i in range(count):
            self.load(i)

    def load(self, i):
        if i % 2:  # from the host or from the device
            self.h.set(i, self.a[i].view(self.torch.int16).numpy(),
                       self.b[i].view(self.torch.int16).numpy(), self.scale[i])
        else:
            self.h.set(i, self.a[i].cuda(), self.b[i].cuda(), self.scale[i], on_device=True)

    def inputs(self, T, x_dtype, y_dtype, mixed=True):
        torch, g = self.torch, self.g
        x = torch.randn(T, self.h.d_in, generator=g).to(dtype_of(torch, x_dtype))
        base = torch.randn(T, self.h.d_out, generator=g).to(dtype_of(torch, y_dtype))
        if mixed:
            ids = torch.randint(-1, self.h.count, (T,), generator=g, dtype=torch.int32)
        else:  # runs of one adapter
            ids = ((torch.arange(T) * 3) // max(T, 3) * 2 % (self.h.count + 1) - 1).int()
        return x, base, ids

    def expect(self, x, base, ids):
        """The definition in 64 bits and the tolerance."""
        x64, y = x.double().numpy(), base.double().numpy().copy()
        S = np.zeros_like(y)
        for t, i in enumerate(ids.tolist()):
            if 0 <= i < self.h.count:
                A, B = self.a[i].double().numpy(), self.b[i].double().numpy()
                y[t] += self.scale[i] * (B @ (A @ x64[t]))
                S[t] = abs(self.scale[i]) * (np.abs(B) @ (np.abs(A) @ np.abs(x64[t])))
        steps = self.h.d_in / 32 + self.h.rank + 48
        tol = steps * HALF * S + 2 * HALF * np.abs(y)
        if base.dtype != self.torch.float32:
            tol += self.torch.finfo(base.dtype).eps / 2 * np.abs(y)
            if base.dtype == self.torch.float16:
                tol += 2.0 ** -25  # half its smallest step
        return y, tol

    def apply(self, x, base, ids, x_dtype, y_dtype, pads=(0, 0, 0), in_place=False, shift=0,
              none=False, stream=None):
        """Runs on copies with rows `pads` elements apart that begin `shift` elements
        behind an aligned address; what lies between and behind the rows stays."""
        torch = self.torch
        T = x.shape[0]

        def wide(v, cols, pad):
            full = torch.full((shift + (T + 1) * (cols + pad),), 7.0, dtype=v.dtype)
            rows = full[shift:].view(T + 1, cols + pad)
            rows[:T, :cols] = v
            return full.cuda()
        xd, bd = wide(x, self.h.d_in, pads[0]), wide(base, self.h.d_out, pads[1])
        idd = ids.cuda()
        pad_y = pads[1] if in_place else pads[2]
        yd = bd if in_place else wide(torch.full_like(base, 5.0), self.h.d_out, pad_y)
        torch.cuda.synchronize()
        size = {torch.float32: 4}.get(base.dtype, 2)
        xsize = {torch.float32: 4}.get(x.dtype, 2)
        self.h.apply(idd, xd.data_ptr() + shift * xsize, yd.data_ptr() + shift * size, T,
                     base=None if none else bd.data_ptr() + shift * size, x_dtype=x_dtype,
                     y_dtype=y_dtype, x_stride=self.h.d_in + pads[0],
                     base_stride=self.h.d_out + pads[1], y_stride=self.h.d_out + pad_y,
                     stream=stream)
        torch.cuda.synchronize()
        out = yd.cpu()[shift:].view(T + 1, -1)
        assert (yd.cpu()[:shift] == 7.0).all()
        assert (out[T] == 7.0).all() and (out[:, self.h.d_out:] == 7.0).all()
        return out[:T, :self.h.d_out]

    def check(self, T, x_dtype, y_dtype, mixed=True, **kw):
        x, base, ids = self.inputs(T, x_dtype, y_dtype, mixed)
        if kw.get("none"):
            base = self.torch.zeros_like(base)
        want, tol = self.expect(x, base, ids)
        got = self.apply(x, base, ids, x_dtype, y_dtype, **kw).double().numpy()
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


def io_types(dtype):
    return [("f32", "f32"), (dtype, dtype), (dtype, "f32"), ("f32", dtype)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("count,rank,d_in,d_out", [
    (1, 1, 1, 1), (3, 4, 64, 64), (5, 16, 4096, 192), (2, 5, 1001, 777), (4, 17, 96, 130),
    (3, 64, 256, 65), (2, 128, 200, 1536), (7, 33, 31, 16), (2, 100, 2048, 40), (3, 8, 8, 8)])
def test_shapes(torch, dtype, count, rank, d_in, d_out):
    s = Setup(torch, count, rank, d_in, d_out, dtype)
    for i, T in enumerate((1, 2, 15, 16, 17, 33, 130)):
        xt, yt = io_types(dtype)[i % 4]
        s.check(T, xt, yt, mixed=i % 2 == 0, in_place=i % 3 == 1, none=i % 3 == 2)
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T", [1, 7, 40, 300, 700])
def test_strides_and_alignment(torch, dtype, T):
    """Rows apart, and rows that begin at addresses of one element only."""
    for rank, d_in, d_out in ((16, 128, 192), (6, 100, 72)):
        s = Setup(torch, 4, rank, d_in, d_out, dtype, seed=T)
        for i, (xt, yt) in enumerate(io_types(dtype)):
            s.check(T, xt, yt, pads=(8, 16, 24), mixed=i % 2 == 0)
            s.check(T, xt, yt, pads=(3, 1, 5), mixed=i % 2 == 1)
            s.check(T, xt, yt, shift=1, in_place=True)
        s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,rank,mixed", [(512, 16, False), (513, 64, True), (2000, 16, False),
                                          (1031, 128, False)])
def test_many_tokens(torch, dtype, T, rank, mixed):
    s = Setup(torch, 9, rank, 320, 448, dtype)
    for xt, yt in io_types(dtype):
        s.check(T, xt, yt, mixed=mixed)
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d_out", [64, 130, 1000, 2048])
@pytest.mark.parametrize("count,rank", [(2, 16), (3, 40), (20, 7)])
def test_tiles_of_several_adapters(torch, dtype, d_out, count, rank):
    """Tiles whose adapters are dealt to the slices of their outputs: fewer slices than
    adapters, as many, more; tokens without one among them, in place too."""
    s = Setup(torch, count, rank, 320, d_out, dtype)
    for i, T in enumerate((257, 400, 1040)):
        xt, yt = io_types(dtype)[(i + rank) % 4]
        s.check(T, xt, yt, mixed=True, in_place=i % 2 == 0, pads=(3, 5, 2))
    x, base, ids = s.inputs(300, "f32", dtype)
    ids[:16], ids[16:32], ids[32:40] = -1, 1, 0  # tiles of none, of one, of some
    want, tol = s.expect(x, base, ids)
    got = s.apply(x, base, ids, "f32", dtype)
    assert (np.abs(got.double().numpy() - want) <= tol).all()
    for at in (33, 200, 299):  # with other neighbours the same bits
        other = torch.where(torch.arange(300) == at, ids, (ids + 1) % count).int()
        assert torch.equal(s.apply(x, base, other, "f32", dtype)[at], got[at])
    s.h.close()


@pytest.mark.gpu
def test_ids_outside_the_table_have_no_adapter(torch):
    s = Setup(torch, 3, 8, 64, 64, "bf16")
    x, base, _ = s.inputs(6, "bf16", "bf16")
    ids = torch.tensor([-1, 3, 2 ** 31 - 1, -2 ** 31, 65536, 1], dtype=torch.int32)
    got = s.apply(x, base, ids, "bf16", "bf16")
    assert torch.equal(got[:5], base[:5])
    want, tol = s.expect(x, base, ids)
    assert (np.abs(got.double().numpy() - want) <= tol).all()
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T", [5, 40, 600])
def test_tokens_do_not_affect_each_other(torch, dtype, T):
    """Infinities and NaN in one token's x and in one adapter's weights stay in the
    rows that use them; every other row keeps its bits."""
    s = Setup(torch, 4, 16, 96, 80, dtype)
    for xt, yt in io_types(dtype):
        x, base, ids = s.inputs(T, xt, yt)
        ids = torch.where(ids == 3, 0, ids).int()
        ids[1], ids[2], ids[3] = 0, 3, 1
        clean = s.apply(x, base, ids, xt, yt)
        s.a[3][:] = float("nan")
        s.b[3][:] = float("inf")
        s.load(3)
        x = x.clone()
        x[1], x[3, 5] = float("inf"), float("nan")
        got = s.apply(x, base, ids, xt, yt)
        kind = {4: torch.int32, 2: torch.int16}[got.element_size()]
        rest = [t for t in range(T) if t not in (1, 2, 3)]
        assert torch.equal(got[rest].view(kind), clean[rest].view(kind))
        for t in (1, 2, 3):
            assert not torch.isfinite(got[t]).all()
        assert torch.isnan(got[3]).all()
        s.a[3], s.b[3] = 0.0, 0.0
        s.load(3)
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rank", [1, 5, 16])
def test_infinities_as_the_formula_has_them(torch, dtype, rank):
    """An infinite x: each output infinite or NaN as in 64 bits, ranks padded or not."""
    s = Setup(torch, 2, rank, 70, 66, dtype)
    for T in (4, 300):
        for xt, yt in io_types(dtype):
            x, base, ids = s.inputs(T, xt, yt)
            ids = ids.clamp(min=0)
            x[:, 7] = float("inf")
            with np.errstate(invalid="ignore"):
                want, _ = s.expect(x, base, ids)
            got = s.apply(x, base, ids, xt, yt).double().numpy()
            assert np.array_equal(np.isnan(got), np.isnan(want))
            assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rank", [3, 24, 60, 128])
def test_fp32_x_of_a_wide_range(torch, dtype, rank):
    """Elements of one row 2^-24 to 2^24, rising, falling and mixed along d_in. In tiles
    fp16 parts of x reach down to 2^-38 of the row's largest (2^-24 of a unit whose 2^14
    it reaches): sum |A| of that on top, through B."""
    s = Setup(torch, 2, rank, 4096 + 40, 70, dtype)
    for T in (6, 300):
        x, base, ids = s.inputs(T, "f32", "f32", mixed=False)
        powers = 2.0 ** torch.linspace(-24, 24, s.h.d_in)
        order = torch.randperm(s.h.d_in, generator=s.g)
        for t in range(T):
            x[t] *= (powers, powers.flip(0), powers[order])[t % 3]
        base = base * 0.0
        want, tol = s.expect(x, base, ids)
        for t, i in enumerate(ids.tolist()):
            if T > 256 and dtype == "f16" and i >= 0:
                A, B = s.a[i].double().abs(), s.b[i].double().abs()
                low = 2.0 ** -38 * x[t].abs().max().item()
                tol[t] += s.scale[i] * low * (B @ A.sum(1)).numpy()
        got = s.apply(x, base, ids, "f32", "f32").double().numpy()
        assert (np.abs(got - want) <= tol).all()
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rank", [1, 20, 50])
def test_fp32_x_with_infinities_among_large_values(torch, dtype, rank):
    """An infinity early or late in a row whose finite values rise to fp32's largest:
    as in 64 bits; a NaN stays with its token."""
    s = Setup(torch, 1, rank, 4096 + 5, 33, dtype)
    for T in (4, 290):
        for at in (3, 2000, 4100):
            x, base, ids = s.inputs(T, "f32", "f32")
            ids = ids * 0
            x *= 2.0 ** torch.linspace(-60, 100, s.h.d_in)
            x[:, at] = float("inf")
            x[1] = torch.randn(s.h.d_in, generator=s.g)  # finite
            x[2] = 0.0
            x[2, at] = float("nan")
            x[3] = 0.0
            with np.errstate(invalid="ignore"):
                want, tol = s.expect(x, base, ids)
            got = s.apply(x, base, ids, "f32", "f32").double().numpy()
            assert np.array_equal(np.isnan(got), np.isnan(want))
            some = np.isfinite(want)
            assert some[1].all() and some[3].all()
            assert np.array_equal(got[~some & ~np.isnan(want)], want[~some & ~np.isnan(want)])
            assert (np.abs(got[some] - want[some]) <= tol[some]).all()
    s.h.close()


@pytest.mark.gpu
def test_offsets_beyond_2_31(torch):
    """Adapters, rows of x and rows of y more than 2^31 elements from the first."""
    h = H.Adapters(4200, 128, 4096, 64, "bf16")  # 2.2e9 elements of A
    g = torch.Generator().manual_seed(1)
    a = (torch.randn(128, 4096, generator=g) / 64).bfloat16()
    b = torch.randn(64, 128, generator=g).bfloat16()
    h.set(4199, a.cuda(), b.cuda(), 1.0, on_device=True)
    step = (1 << 31) + 8
    x, y = torch.randn(2, 4096, generator=g).bfloat16(), torch.empty(2, 64)
    buf = torch.empty(step + 4096, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(step + 64, dtype=torch.bfloat16, device="cuda")
    buf[:4096], buf[step:] = x[0].cuda(), x[1].cuda()
    for ids in ([4199, 4199], [0, 4199]):
        h.apply(torch.tensor(ids, dtype=torch.int32).cuda(), buf, out, 2, x_stride=step,
                y_stride=step)
        torch.cuda.synchronize()
        y[0], y[1] = out[:64].cpu().float(), out[step:].cpu().float()
        u = x.double() @ a.double().t()
        want = u @ b.double().t()
        S = (x.double().abs() @ a.double().abs().t()) @ b.double().abs().t()
        tol = (4096 / 32 + 128 + 48) * HALF * S + 2.0 ** -8 * want.abs()
        if ids[0] == 0:
            want[0], tol[0] = 0.0, 0.0
        assert ((y.double() - want).abs() <= tol).all()
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_wide_range(torch, dtype):
    """Rows of very large and very small values: u keeps fp32's range between the
    two products, whatever the weights' type holds."""
    s = Setup(torch, 2, 16, 128, 64, dtype)
    for T in (3, 64, 512):
        x, base, ids = s.inputs(T, "f32", "f32")
        x = x * torch.logspace(-25, 25, T)[:, None]
        base = base * 0.0
        want, tol = s.expect(x, base, ids)
        got = s.apply(x, base, ids, "f32", "f32").double().numpy()
        assert (np.abs(got - want) <= tol + 2.0 ** -126).all()
    if dtype == "f16":  # products above fp16's largest value, brought back by B
        s.a[:] = 60.0
        s.b[:] = s.b * 2.0 ** -12
        for i in range(2):
            s.load(i)
        for T in (3, 64, 512):
            x, base, ids = s.inputs(T, "f16", "f16")
            x = x.abs() * 20.0
            want, tol = s.expect(x, base, ids)
            got = s.apply(x, base, ids, "f16", "f16").double().numpy()
            assert (np.abs(got - want) <= tol).all()
    s.h.close()


@pytest.mark.gpu
def test_an_adapter_is_zero_until_set_and_replaced_by_set(torch):
    h = H.Adapters(2, 4, 32, 48, "f16")
    x, base = torch.randn(3, 32).half().cuda(), torch.randn(3, 48).half().cuda()
    ids, y = torch.tensor([0, 1, 0], dtype=torch.int32).cuda(), torch.empty_like(base)
    h.apply(ids, x, y, 3, base=base)
    torch.cuda.synchronize()
    assert torch.equal(y, base)
    for k in (1.0, 3.0):
        a, b = torch.full((4, 32), k).half().cuda(), torch.full((48, 4), 0.25).half().cuda()
        h.set(1, a, b, 2.0, on_device=True)
        h.apply(ids, x, y, 3, base=None, y_dtype="f16")
        torch.cuda.synchronize()
        want = 2.0 * k * x[1].double().sum().item()
        assert (y[0] == 0).all() and (y[2] == 0).all()
        # 32 sums and 4, one rounding to fp16
        tol = 64 * HALF * 2 * k * x[1].double().abs().sum().item() + 2.0 ** -11 * abs(want)
        assert (y[1].double() - want).abs().max().item() <= tol
    h.close()


@pytest.mark.gpu
def test_apply_refusals(torch):
    h = H.Adapters(2, 8, 64, 96, "bf16")
    lib = H.lib()
    buf = torch.zeros(1 << 14, device="cuda")
    p = buf.data_ptr()
    ids, x, y = p, p + 4096, p + 32768

    def call(ids=ids, x=x, xt=2, xs=64, base=None, bs=96, y=y, yt=2, ys=96, T=4):
        return lib.hy3x_adapters_apply(h._h, ids, x, xt, xs, base, bs, y, yt, ys, T, None)
    assert call() == 0 and call(T=0, ids=None, x=None, y=None) == 0
    for bad in (dict(xt=1), dict(yt=1), dict(xt=5), dict(T=-1), dict(T=(1 << 24) + 1), dict(xs=63),
                dict(ys=95), dict(base=y, bs=95), dict(xs=1 << 33), dict(ids=None), dict(x=None),
                dict(y=None), dict(ids=p + 2), dict(x=x + 1), dict(y=y + 1, yt=2),
                dict(y=y + 2, yt=0), dict(base=y + 2), dict(base=y - 2), dict(base=y, bs=98),
                dict(x=y), dict(x=y + 2 * 96 * 4 - 2), dict(y=x + 2 * 64 * 4 - 2)):
        assert call(**bad) == -1, bad
        assert lib.hy3x_last_error()
    # rows of one wider buffer between each other, and the base itself
    assert call(x=y + 2 * 96, xs=160, ys=160) == 0
    assert call(x=y + 2 * 95, xs=160, ys=160) == -1
    assert call(x=y - 2 * 64, xs=160, ys=160) == 0
    assert call(x=y - 2 * 63, xs=160, ys=160) == -1
    assert call(base=y) == 0
    assert lib.hy3x_adapters_set(h._h, 2, p, p, 1.0, 1) == -1
    assert lib.hy3x_adapters_set(h._h, 0, None, p, 1.0, 1) == -1
    torch.cuda.synchronize()
    h.close()


@pytest.mark.gpu
def test_y_on_its_ids_is_refused(torch):
    h = H.Adapters(2, 8, 64, 96, "bf16")
    buf = torch.zeros(1 << 14, device="cuda")
    y = buf.data_ptr() + 8192

    def call(ids, T=4):
        return H.lib().hy3x_adapters_apply(h._h, ids, y + 32768, 2, 64, None, 96, y, 2, 96, T, None)
    for ids in (y, y - 12, y + 4 * 96 * 2 - 4):
        assert call(ids) == -1 and b"ids" in H.lib().hy3x_last_error()
    assert call(y - 16) == 0 and call(y + 4 * 96 * 2) == 0
    torch.cuda.synchronize()
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("io", ["same", "f32"])
def test_types_of_tensors(torch, io):
    s = Setup(torch, 2, 8, 64, 96, "f16")
    t = torch.float32 if io == "f32" else torch.float16
    x = torch.randn(3, 64, generator=s.g).to(t).cuda()
    ids = torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda")
    y, named = (torch.zeros(3, 96, dtype=t, device="cuda") for _ in range(2))
    kind = "f32" if io == "f32" else "f16"
    s.h.apply(ids, x, named, 3, x_dtype=kind, y_dtype=kind)
    s.h.apply(ids, x, y, 3)  # the tensors' own types
    torch.cuda.synchronize()
    assert torch.equal(y, named) and y.abs().max() > 0
    with pytest.raises(H.HY3XError, match="type"):
        s.h.apply(ids, x.bfloat16(), y, 3)
    for bad in (dict(ids=ids.long()), dict(x=x.double()), dict(y=y.double()),
                dict(base=y.bfloat16())):
        with pytest.raises(TypeError):
            s.h.apply(**dict(dict(ids=ids, x=x, y=y, T=3), **bad))
    with pytest.raises(AssertionError):
        s.h.set(0, torch.zeros(8, 64, device="cuda"), torch.zeros(96, 8, device="cuda"),
                on_device=True)
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 600])
def test_streams_and_graph(torch, T):
    """Two calls of one handle at once, and a captured one replayed on new inputs."""
    s = Setup(torch, 5, 16, 256, 320, "bf16")
    sets = [s.inputs(T, "bf16", "bf16") for _ in range(2)]
    want = [s.apply(x, base, ids, "bf16", "bf16") for x, base, ids in sets]
    dev = [[v.cuda() for v in one] for one in sets]
    ys = [torch.zeros_like(d[1]) for d in dev]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for d, y, st in zip(dev, ys, streams):
        s.h.apply(d[2], d[0], y, T, base=d[1], stream=st.cuda_stream)
    torch.cuda.synchronize()
    for y, w in zip(ys, want):
        assert torch.equal(y.cpu(), w)
    x, base, ids = (v.clone() for v in dev[0])
    y = torch.zeros_like(base)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.h.apply(ids, x, y, T, base=base, stream=torch.cuda.current_stream().cuda_stream)
    for i in (1, 0, 1):
        for d, src in zip((x, base, ids), dev[i]):
            d.copy_(src)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), want[i])
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T", [1, 60, 300])
@pytest.mark.parametrize("rank,d_in", [(2, 2), (5, 40), (64, 200), (128, 33)])
def test_all_bits_of_the_product_reach_y(torch, dtype, T, rank, d_in):
    """One rank's u is x[0] = 1 + 2^-11 + (4 j + 3) 2^-23, all 24 bits of fp32, another's 1.
    B of 1 and -2^-11 and a base of -1 leave the lowest bits, which y's type holds: every
    sum is a multiple of 2^-23 below 2, so every step is exact, and y too."""
    t = dtype_of(torch, dtype)
    h = H.Adapters(1, rank, d_in, 70, dtype)
    a, b = torch.zeros(rank, d_in, dtype=t), torch.zeros(70, rank, dtype=t)
    a[0, 0], a[rank - 1, 1] = 1.0, 1.0
    b[:, 0], b[:, rank - 1] = 1.0, -2.0 ** -11
    h.set(0, a.cuda(), b.cuda(), 1.0, on_device=True)
    low = (4.0 * (torch.arange(T) % 61) + 3.0) * 2.0 ** -23  # 8 bits
    x = torch.zeros(T, d_in)
    x[:, 0], x[:, 1] = 1.0 + 2.0 ** -11 + low, 1.0
    ids, base = torch.zeros(T, dtype=torch.int32).cuda(), torch.full((T, 70), -1.0, dtype=t).cuda()
    y = torch.zeros_like(base)
    h.apply(ids, x.cuda(), y, T, base=base)
    torch.cuda.synchronize()
    assert torch.equal(y.float().cpu(), low[:, None].expand(T, 70))
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T", [3, 300])
def test_a_token_without_an_adapter_keeps_its_base(torch, dtype, T):
    """Bit for bit: zeros of either sign, infinities, the smallest and the largest; 0
    where there is no base."""
    s = Setup(torch, 2, 8, 64, 72, dtype)
    for xt, yt in io_types(dtype):
        x, base, _ = s.inputs(T, xt, yt)
        info = torch.finfo(base.dtype)
        base[:, ::8], base[:, 1::8], base[:, 2::8] = -0.0, 0.0, float("-inf")
        base[:, 3::8], base[:, 4::8], base[:, 5::8] = info.max, info.min, info.smallest_normal
        ids = torch.full((T,), -1, dtype=torch.int32)
        kind = {4: torch.int32, 2: torch.int16}[base.element_size()]
        for i in ([], [1], list(range(0, T, 2))):  # alone, and beside tokens with one
            ids[i] = 1
            got = s.apply(x, base, ids, xt, yt)
            rest = [t for t in range(T) if ids[t] < 0]
            assert torch.equal(got[rest].view(kind), base[rest].view(kind))
            none = s.apply(x, base, ids, xt, yt, none=True)
            assert (none[rest].view(kind) == 0).all()
    s.h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T", [5, 256, 257])
@pytest.mark.parametrize("rank", [1, 20, 128])
def test_infinite_weights(torch, dtype, T, rank):
    """An infinite or NaN element of B makes its own output so, one of A every output of
    its adapter's tokens, whether by infinity or NaN; all others are as they should be."""
    s = Setup(torch, 3, rank, 70, 66, dtype)
    inf, nan = float("inf"), float("nan")
    s.b[0, 9, rank - 1], s.b[0, 65, 0], s.b[0, 30, 0] = inf, -inf, nan
    s.a[1, rank - 1, 69] = inf
    for i in (0, 1):
        s.load(i)
    for xt, yt in io_types(dtype):
        x, base, ids = s.inputs(T, xt, yt)
        ids[0], ids[1], ids[2] = 0, 1, 2
        x[3:] = x[3:].round()  # zeros among them: 0 inf is NaN in any arithmetic
        with np.errstate(invalid="ignore"):
            want, tol = s.expect(x, base, ids)
        got = s.apply(x, base, ids, xt, yt).double().numpy()
        fine = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), fine)
        assert (~fine[0]).sum() == 3 and not fine[1].any() and fine[2].all()
        assert (np.abs(got[fine] - want[fine]) <= tol[fine]).all()
    s.h.close()
