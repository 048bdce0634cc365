"""hy3x_linear4_*: products of 4-bit weights with group scales, against the definition in
64 bits.

Tolerance of an output, in steps of 2^-24 of A = sum_k |x| s (q + z), which bounds every
partial sum: an output's sum passes at most two additions for each weight of a group (q x
and z x), one for each group and 32 where waves and parts are joined; then the base's
addition and the rounding to y's type, at most half a step of the value."""
import ctypes

import numpy as np
import pytest

import hy3_amd as H

HALF = 2.0 ** -24
RNG = np.random.default_rng


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


# ---------------------------------------------------------------- refusals (no GPU)
def test_create_refusals():
    lib, h = H.lib(), ctypes.c_void_p()
    good = dict(d_out=64, d_in=96, group=32, type=2)
    for bad, word in ((dict(d_out=0), b"d_out"), (dict(d_out=(1 << 20) + 1), b"d_out"),
                      (dict(d_in=7), b"d_in"), (dict(d_in=65537), b"d_in"),
                      (dict(group=0), b"group"), (dict(group=48), b"group"),
                      (dict(group=256), b"group"), (dict(type=0), b"type"),
                      (dict(type=3), b"type")):
        v = dict(good, **bad)
        assert lib.hy3x_linear4_create(ctypes.byref(h), v["d_out"], v["d_in"], v["group"],
                                       v["type"]) == -1, bad
        assert word in lib.hy3x_last_error() and not h.value
    assert lib.hy3x_linear4_create(None, 64, 96, 32, 2) == -1
    assert lib.hy3x_linear4_set(None, 4096, 4096, None, 0) == -1
    assert lib.hy3x_linear4_apply(None, 4096, 0, 64, None, 0, 8192, 0, 64, 1, None) == -1
    assert lib.hy3x_linear4_destroy(None) == 0


# ---------------------------------------------------------------- the definition
def make(d_out, d_in, group, scale_type, zeros, seed, torch):
    """q [d_out x d_in], scales and zeros on the CPU, and the packed bytes."""
    g = torch.Generator().manual_seed(seed)
    groups = -(-d_in // group)
    q = torch.randint(0, 16, (d_out, d_in), generator=g, dtype=torch.uint8)
    s = (0.01 * torch.exp(0.5 * torch.randn(d_out, groups, generator=g))).to(scale_type)
    z = torch.randint(0, 17, (d_out, groups), generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z, pack(q, torch)


def pack(q, torch):
    if q.shape[1] % 2:  # the last byte's high half is nobody's: anything
        q = torch.cat((q, torch.full_like(q[:, :1], 11)), 1)
    return (q[:, 0::2] | q[:, 1::2] << 4).contiguous()


def held(d_out, d_in, group, name, q, s, z, packed):
    h = H.Linear4(d_out, d_in, group=group, dtype=name)
    h.set(packed.cuda(), s.cuda(), None if z is None else z.cuda(), on_device=True)
    return h


def definition(q, s, z, group, x, base, torch):
    """y and A = sum |x| s (q + z), in 64 bits."""
    of = torch.arange(q.shape[1]) // group
    zd = torch.full(s.shape, 8.0, dtype=torch.float64) if z is None else z.double()
    sd, qd, xd = s.double()[:, of], q.double(), x.double().cpu()
    y = xd @ ((qd - zd[:, of]) * sd).t()
    a = xd.abs() @ ((qd + zd[:, of]) * sd.abs()).t()
    if base is not None:
        y = y + base.double().cpu()
    return y, a


def check(y, exact, a, d_in, group, base, torch):
    steps = 2 * min(group, d_in) + -(-d_in // group) + 32
    tol = steps * HALF * a + torch.finfo(y.dtype).eps / 2 * exact.abs() + 1e-40
    if y.dtype == torch.float16:
        tol += 2.0 ** -25  # half a step of its smallest numbers
    if base is not None:
        tol += HALF * (exact.abs() + base.double().cpu().abs())
    far = (y.double().cpu() - exact).abs()
    worst = (far / tol).max().item()
    assert worst <= 1.0, (worst, (far > tol).nonzero()[:5].tolist())


def run_case(torch, T, d_in, d_out, group=128, scales="bf16", zeros=False, x="bf16", y="bf16",
             base=None, pad=0, at=0, seed=1):
    """pad: elements between rows of x, y and base; at: elements before the first."""
    types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    q, s, z, packed = make(d_out, d_in, group, types[scales], zeros, seed, torch)
    h = held(d_out, d_in, group, scales, q, s, z, packed)
    g = torch.Generator().manual_seed(seed + 1)

    def rows(width, kind):
        flat = torch.randn(T * (width + pad) + at, generator=g).to(types[kind]).cuda()
        return flat, flat[at:].view(T, width + pad)[:, :width]
    _, xs = rows(d_in, x)
    flat, ys = rows(d_out, y)
    b = None
    if base == "own":
        b = rows(d_out, y)[1]
    elif base == "y":
        b = ys
    b0 = None if b is None else b.clone()
    before = flat.clone()
    h.apply(xs, ys, T, base=b)
    torch.cuda.synchronize()
    exact, a = definition(q, s, z, group, xs, b0, torch)
    check(ys, exact, a, d_in, group, b0, torch)
    # nothing but the rows is written
    ys.copy_(before[at:].view(T, d_out + pad)[:, :d_out])
    assert torch.equal(flat, before)
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T", [1, 2, 4, 5, 15, 16, 17, 31, 33, 48, 64, 65, 100, 129, 257])
def test_tokens(torch, T, x):
    run_case(torch, T, 640, 200, x=x, y=x, zeros=T % 2 == 0, scales="f16" if T % 3 else "bf16",
             group=(32, 64, 128)[T % 3])


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("d_in", [8, 9, 15, 31, 33, 64, 127, 128, 130, 511, 512, 513, 1001, 2049])
def test_inputs(torch, d_in, group):
    for T, x in ((1, "bf16"), (3, "f32"), (20, "f16"), (70, "bf16"), (130, "f32")):
        run_case(torch, T, d_in, 33, group=group, x=x, y="f32", zeros=T != 3, seed=d_in)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6, 40, 150])
@pytest.mark.parametrize("d_out", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 1000])
def test_outputs(torch, d_out, T):
    run_case(torch, T, 257, d_out, x="f16", y="f16", scales="f16", zeros=True, group=64)
    run_case(torch, T, 384, d_out, x="f32", y="bf16", base="own")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 16, 30, 64, 200])
@pytest.mark.parametrize("d_in", [4096, 4224, 8192, 9000, 13312, 17000])
def test_long_rows(torch, d_in, T):
    run_case(torch, T, d_in, 80, x="bf16", y="f32", zeros=True)
    run_case(torch, T, d_in, 80, x="f32", y="f32", group=32, scales="f16")


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("y", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("base", [None, "own", "y"])
def test_types_bases_and_strides(torch, x, y, base):
    for T, pad, at in ((1, 0, 0), (1, 0, 1), (9, 3, 1), (40, 8, 8), (70, 1, 5), (150, 5, 3)):
        run_case(torch, T, 200, 100, group=64, x=x, y=y, base=base, pad=pad, at=at,
                 scales="f16" if pad else "bf16", zeros=T == 9)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 5, 16, 17, 48, 64, 65, 130, 300])
def test_many_outputs(torch, T):
    """More row tiles than blocks take at once."""
    run_case(torch, T, 300, 20011, x="bf16", y="f32", zeros=True, group=64)
    run_case(torch, T, 1100, 9000, x="f32", y="f32")


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T", [1, 5, 16, 40, 64, 150, 500])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_whole_numbers_are_exact(torch, T, x, group):
    """Small integers x, scales that are powers of two: every sum is a whole number below
    2^24, so that no weight may be off, and none counted twice."""
    types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    d_out, d_in = 150, 900
    q, s, z, packed = make(d_out, d_in, group, torch.bfloat16, True, 7, torch)
    g = torch.Generator().manual_seed(T)
    s = (2.0 ** torch.randint(0, 3, s.shape, generator=g)).to(torch.bfloat16)
    h = held(d_out, d_in, group, "bf16", q, s, z, packed)
    xs = torch.randint(-8, 9, (T, d_in), generator=g).to(types[x]).cuda()
    y = torch.full((T, d_out), 5.0, device="cuda")
    h.apply(xs, y, T)
    exact, _ = definition(q, s, z, group, xs, None, torch)
    assert torch.equal(y.cpu().double(), exact)
    h.apply(xs, y, T, base=y)
    assert torch.equal(y.cpu().double(), 2 * exact)
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 33, 130])
def test_wide_values(torch, T):
    """Activations over the whole range of their type, fp16's smallest among them."""
    for kind, low, high in ((torch.float16, -24, 10), (torch.bfloat16, -100, 40),
                            (torch.float32, -90, 40)):
        q, s, z, packed = make(70, 260, 64, torch.float16, True, 3, torch)
        h = held(70, 260, 64, "f16", q, s, z, packed)
        g = torch.Generator().manual_seed(T)
        x = torch.randn(T, 260, generator=g) * 2.0 ** torch.randint(low, high, (T, 1), generator=g)
        x = x.to(kind).cuda()
        y = torch.empty(T, 70, device="cuda")
        h.apply(x, y, T)
        exact, a = definition(q, s, z, 64, x, None, torch)
        check(y, exact, a, 260, 64, None, torch)
        h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T", [2, 16, 20, 64, 200])
def test_a_token_keeps_its_infinities(torch, T, x):
    types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    q, s, z, packed = make(90, 300, 32, torch.bfloat16, True, 5, torch)
    h = held(90, 300, 32, "bf16", q, s, z, packed)
    xs = torch.randn(T, 300, generator=torch.Generator().manual_seed(2)).to(types[x]).cuda()
    clean = torch.empty(T, 90, device="cuda")
    h.apply(xs, clean, T)
    for value in (float("inf"), float("-inf"), float("nan")):
        bad = xs.clone()
        bad[T // 2, 299] = value
        y = torch.empty_like(clean)
        h.apply(bad, y, T)
        assert not y[T // 2].isfinite().any()
        y[T // 2] = clean[T // 2]
        assert torch.equal(y, clean)
    h.close()


@pytest.mark.gpu
def test_results_do_not_depend_on_the_rest_of_the_batch(torch):
    """Twice the same bits; and in a batch of the same path a token's own."""
    q, s, z, packed = make(200, 700, 64, torch.bfloat16, True, 5, torch)
    h = held(200, 700, 64, "bf16", q, s, z, packed)
    for T in (7, 16, 64, 300):
        x = torch.randn(T, 700, generator=torch.Generator().manual_seed(T)).bfloat16().cuda()
        a, b = torch.empty(T, 200, device="cuda"), torch.empty(T, 200, device="cuda")
        h.apply(x, a, T)
        h.apply(x, b, T)
        assert torch.equal(a, b)
        h.apply(x.flip(0).contiguous(), b, T)
        assert torch.equal(a, b.flip(0))
    h.close()


@pytest.mark.gpu
def test_host_weights_and_again(torch):
    """Set from host arrays, and set again: with other zero points, and without."""
    q, s, z, packed = make(50, 130, 32, torch.float16, True, 5, torch)
    h = H.Linear4(50, 130, group=32, dtype="f16")
    x = torch.randn(3, 130, generator=torch.Generator().manual_seed(2)).half().cuda()
    y = torch.empty(3, 50, device="cuda")
    with pytest.raises(H.HY3XError, match="not set"):
        h.apply(x, y, 3)
    for scales in (s.numpy(), s.view(torch.int16).numpy()):
        for zz in (z, None):
            h.set(packed.numpy(), scales, None if zz is None else zz.numpy())
            h.apply(x, y, 3)
            exact, a = definition(q, s, zz, 32, x, None, torch)
            check(y, exact, a, 130, 32, None, torch)
    kept = y.clone()
    bad = z.clone()
    bad[49, 4] = 17
    for args in ((packed.numpy(), s.numpy(), bad.numpy()),
                 (packed.cuda(), s.cuda(), bad.cuda(), True)):
        with pytest.raises(H.HY3XError, match="above 16"):
            h.set(*args)
    h.apply(x, y, 3)
    assert torch.equal(y, kept)
    h.close()


@pytest.mark.gpu
def test_argument_refusals(torch):
    lib = H.lib()
    h = H.Linear4(64, 96, group=32, dtype="bf16")
    x = torch.zeros(8, 96, dtype=torch.bfloat16, device="cuda")
    assert lib.hy3x_linear4_set(h._h, None, 4096, None, 1) == -1
    assert lib.hy3x_linear4_set(h._h, 4096, None, None, 1) == -1
    assert lib.hy3x_linear4_set(h._h, 4096, 4097, None, 1) == -1
    h.set(torch.zeros(64, 48, dtype=torch.uint8, device="cuda"),
          torch.ones(64, 3, dtype=torch.bfloat16, device="cuda"), on_device=True)
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    y, b = buf.data_ptr() + 8192, buf.data_ptr() + 32768
    good = dict(x=x.data_ptr(), x_type=2, x_stride=96, base=None, base_stride=0, y=y, y_type=0,
                y_stride=64, T=8)

    def call(**change):
        v = dict(good, **change)
        return lib.hy3x_linear4_apply(h._h, *(v[k] for k in good), None)
    assert call() == 0 and call(T=0, x=None, y=None) == 0
    assert call(base=y, base_stride=64) == 0 and call(base=b, base_stride=64) == 0
    for bad in (dict(x=None), dict(y=None), dict(x_type=3), dict(x_type=-1), dict(y_type=3),
                dict(x_stride=95), dict(y_stride=63), dict(base=b, base_stride=63),
                dict(x_stride=(1 << 32) + 1), dict(T=-1), dict(T=(1 << 24) + 1),
                dict(x=x.data_ptr() + 1), dict(y=y + 2), dict(base=b + 2, base_stride=64),
                dict(base=y + 4, base_stride=64), dict(base=y, base_stride=65),
                dict(x=y, x_type=0), dict(x=y + 64 * 4 * 8 - 4)):
        assert call(**bad) == -1, bad
    torch.cuda.synchronize()
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 40, 200])
def test_graph_and_streams(torch, T):
    """Captured and replayed with other inputs, eager work between; and two calls at once."""
    q, s, z, packed = make(300, 520, 128, torch.bfloat16, True, 5, torch)
    h = held(300, 520, 128, "bf16", q, s, z, packed)
    x = torch.randn(4, T, 520, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    want = torch.empty(4, T, 300, device="cuda")
    for i in range(4):
        h.apply(x[i], want[i], T)
    torch.cuda.synchronize()
    into, out = x[0].clone(), torch.empty(T, 300, device="cuda")
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        h.apply(into, out, T, stream=torch.cuda.current_stream().cuda_stream)
    for i in (1, 3, 0, 2):
        into.copy_(x[i])
        out.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = torch.zeros_like(want)
    torch.cuda.synchronize()
    for _ in range(5):
        for i, st in enumerate(streams):
            h.apply(x[i], got[i], T, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    h.close()


@pytest.mark.gpu
def test_far_rows(torch):
    """Rows whose elements lie past 32-bit offsets."""
    q, s, z, packed = make(40, 200, 64, torch.bfloat16, True, 5, torch)
    h = held(40, 200, 64, "bf16", q, s, z, packed)
    far = (1 << 31) + 8
    room = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device="cuda")
    for T in (3, 3 * 8):  # the first three rows lie far apart, the path's other rows follow
        stride = far if T == 3 else far // 8
        x = torch.as_strided(room, (T, 200), (stride, 1)) if T == 3 else \
            torch.as_strided(room, (16, 200), (stride, 1))
        n = x.shape[0]
        x.copy_(torch.randn(n, 200, generator=torch.Generator().manual_seed(2)))
        y = torch.empty(n, 40, device="cuda")
        h.apply(x, y, n)
        exact, a = definition(q, s, z, 64, x, None, torch)
        check(y, exact, a, 200, 64, None, torch)
        dense = x.contiguous()
        out = torch.as_strided(room, (n, 40), (stride, 1), 2048)
        h.apply(dense, out, n)
        exact, a = definition(q, s, z, 64, dense, None, torch)
        check(out, exact, a, 200, 64, None, torch)
    h.close()


@pytest.mark.gpu
def test_many_weights(torch):
    """A matrix whose bytes pass 2^31: its last rows."""
    d_out, d_in = 1 << 17, 40000
    h = H.Linear4(d_out, d_in, group=128, dtype="bf16")
    g = torch.Generator(device="cuda").manual_seed(3)
    packed = torch.randint(0, 256, (d_out, d_in // 2), generator=g, dtype=torch.uint8,
                           device="cuda")
    s = 0.01 * torch.rand(d_out, 313, generator=g, device="cuda")
    s = s.bfloat16()
    h.set(packed, s, on_device=True)
    tail = slice(d_out - 100, d_out)
    p = packed[tail].cpu()
    q = torch.stack((p & 15, p >> 4), 2).view(100, -1)
    for T in (1, 20, 70):
        x = torch.randn(T, d_in, generator=g, device="cuda").bfloat16()
        y = torch.empty(T, d_out, device="cuda")
        h.apply(x, y, T)
        exact, a = definition(q, s[tail].cpu(), None, 128, x, None, torch)
        check(y[:, tail], exact, a, d_in, 128, None, torch)
    h.close()


@pytest.mark.gpu
def test_most_weights(torch):
    """More weights than a launch has threads to lay them out: its first and last rows."""
    d_out, d_in = 1 << 20, 32776
    torch.cuda.empty_cache()
    g = torch.Generator(device="cuda").manual_seed(3)
    packed = torch.randint(0, 256, (d_out, d_in // 2), generator=g, dtype=torch.uint8,
                           device="cuda")
    s = (0.01 * torch.rand(d_out, 257, generator=g, device="cuda")).bfloat16()
    h = H.Linear4(d_out, d_in, group=128, dtype="bf16")
    h.set(packed, s, on_device=True)
    rows = torch.cat((torch.arange(50), torch.arange(d_out - 50, d_out)))
    p = packed[rows.cuda()].cpu()
    q = torch.stack((p & 15, p >> 4), 2).view(100, -1)
    for T in (1, 20):
        x = torch.randn(T, d_in, generator=g, device="cuda").bfloat16()
        y = torch.empty(T, d_out, device="cuda")
        h.apply(x, y, T)
        exact, a = definition(q, s[rows.cuda()].cpu(), None, 128, x, None, torch)
        check(y[:, rows.cuda()], exact, a, d_in, 128, None, torch)
    h.close()


@pytest.mark.gpu
def test_most_outputs(torch):
    """More outputs than a launch has threads for: a second one has the last tokens."""
    T, d_out = 4194300, 1 << 14
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 145 << 30:
        pytest.skip("needs 145 GB of free device memory")
    q, s, z, packed = make(d_out, 8, 32, torch.bfloat16, True, 5, torch)
    h = held(d_out, 8, 32, "bf16", q, s, z, packed)
    x = torch.randn(T, 8, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    y = torch.empty(T, d_out, dtype=torch.bfloat16, device="cuda")
    h.apply(x, y, T)
    torch.cuda.synchronize()
    for at in (0, T // 2, T - 40, T - 8):
        n = slice(at, at + 8)
        exact, a = definition(q, s, z, 32, x[n], None, torch)
        check(y[n], exact, a, 8, 32, None, torch)
    del y
    torch.cuda.empty_cache()
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
def test_weights_set_again_after_a_capture(torch, T):
    """A replay reads the weights set last; where that cannot be, they are refused."""
    first = make(100, 1300, 64, torch.bfloat16, True, 5, torch)
    other = make(100, 1300, 64, torch.bfloat16, True, 6, torch)
    x = torch.randn(T, 1300, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    for zeros in (True, False):
        q, s, z, packed = first
        h = held(100, 1300, 64, "bf16", q, s, z if zeros else None, packed)
        y = torch.empty(T, 100, device="cuda")
        h.apply(x, y, T)
        st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            h.apply(x, y, T, stream=torch.cuda.current_stream().cuda_stream)
        q, s, z, packed = other
        for zz in ((z, None, z) if zeros else (None,)):
            h.set(packed.cuda(), s.cuda(), None if zz is None else zz.cuda(), on_device=True)
            for _ in range(2):
                y.fill_(-1.0)
                graph.replay()
                torch.cuda.synchronize()
                exact, a = definition(q, s, zz, 64, x, None, torch)
                check(y, exact, a, 1300, 64, None, torch)
        if not zeros:
            kept = y.clone()
            with pytest.raises(H.HY3XError, match="captured"):
                h.set(packed.cuda(), s.cuda(), z.cuda(), on_device=True)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, kept)
        h.close()


# one of each path: x in registers (all tiles at once; streams of weights, with one and two
# quads a wave), then the shapes of tiles through LDS, by tokens, inputs and outputs
SHAPES = [(1, 7000, 4000), (4, 512, 5000), (16, 4000, 4000), (11, 8192, 900),
          (1, 2500, 20000), (3, 4096, 20000), (16, 3900, 20000), (9, 2560, 17000),
          (4, 8192, 9000), (2, 5000, 9000), (1, 6400, 12600),
          (9, 1152, 33000), (16, 1152, 13000), (9, 3200, 7000), (13, 8320, 1000), (3, 8448, 70),
          (20, 256, 5000), (20, 6272, 500), (33, 384, 12000), (50, 256, 13000),
          (130, 256, 8000), (130, 256, 12000), (170, 256, 14000), (40, 256, 10000),
          (100, 3200, 7500), (300, 3200, 4000), (30, 256, 110000), (200, 256, 20000), (60, 128, 60000),
          (500, 256, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,d_in,d_out", SHAPES)
def test_every_shape_is_exact(torch, T, d_in, d_out, group, x):
    """Small integers x, scales 1/2, 1 and 2: every sum is below 2^24 halves, so that fp32
    sums in any order are exact. Rows of whole chunks, aligned to 16 bytes, and others."""
    kind = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[x]
    g = torch.Generator(device="cuda").manual_seed(T + d_in)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda")
    for n in {d_in // 128 * 128, d_in - 21}:
        packed = whole(0, 256, d_out, (n + 1) // 2).to(torch.uint8)
        groups = -(-n // group)
        z = whole(0, 17, d_out, groups).to(torch.uint8)
        s = (2.0 ** (whole(0, 3, d_out, groups) - 1)).bfloat16()
        xs = whole(-8, 9, T, n + 8).to(kind)[:, :n]
        of = torch.arange(n, device="cuda") // group
        q = torch.stack((packed & 15, packed >> 4), 2).view(d_out, -1)[:, :n]
        w = (q.float() - z.float()[:, of]) * s.float()[:, of]
        want = xs.float() @ w.t()
        h = H.Linear4(d_out, n, group=group, dtype="bf16")
        h.set(packed, s, z, on_device=True)
        y = torch.full((T, d_out), 5.0, device="cuda")
        h.apply(xs, y, T)
        assert torch.equal(y, want), (n, (y != want).nonzero()[:5].tolist())
        if n % 128 == 0 and T > 1:  # rows at odd elements
            h.apply(xs[1:], y, T - 1, x_stride=n + 8)
            assert torch.equal(y[:T - 1], want[1:])
            odd = torch.empty(T * (n + 1) + 1, dtype=kind, device="cuda")[1:].view(T, n + 1)[:, :n]
            odd.copy_(xs)
            y.fill_(5.0)
            h.apply(odd, y, T)
            assert torch.equal(y, want)
        h.close()
