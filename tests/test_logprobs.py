"""hy3x_logprobs against the definition in 64 bits.

Ids have to be equal. With d = l - max l of a row, p = softmax, and 2^-24 the relative
error of a rounding in fp32: an exponential is off by (2 |d| + 4) of them (d itself, its
product with log2 e, the exponential's last step), a sum over a row by its additions in
fp32, at most V / 256 + 8 of them before the parts meet in 64 bits. So log S is off by
n + 2 E|d| of them, E the mean under p; a log-probability by that and one rounding of
its value; the entropy by n (1 + E|d|) + 2 E|d| + 3 E d^2 and the rounding of its value."""
import ctypes

import numpy as np
import pytest

import hy3_amd as H

HALF = 2.0 ** -24
NAMES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


# ---------------------------------------------------------------- refusals (no GPU)
def test_workspace_refusals():
    lib = H.lib()
    assert lib.hy3x_logprobs_workspace(0, 1, 0) == 0
    for bad in ((-1, 10, 0), (1, 0, 0), (1, (1 << 24) + 1, 0), ((1 << 24) + 1, 10, 0),
                (1, 10, -1), (1, 100, 33), (1, 3, 4)):
        assert lib.hy3x_logprobs_workspace(*bad) == -1, bad
        with pytest.raises(H.HY3XError):
            H.logprobs_workspace(*bad)


def test_argument_refusals():
    lib = H.lib()
    good = dict(logits=1 << 20, type=0, stride=1000, V=1000, tokens=4096, T=4, top=5, logp=8192,
                entropy=12288, ids=16384, lp=20480, ws=1 << 24, room=1 << 24)

    def call(**change):
        v = dict(good, **change)
        return lib.hy3x_logprobs(*(v[k] for k in good), None)
    for bad in (dict(logits=None), dict(type=3), dict(type=-1), dict(stride=999),
                dict(stride=(1 << 32) + 1), dict(V=0), dict(V=(1 << 24) + 1), dict(tokens=None),
                dict(T=-1), dict(T=(1 << 24) + 1), dict(top=-1), dict(top=33), dict(logp=None),
                dict(V=4), dict(ids=None), dict(lp=None), dict(logits=(1 << 20) + 2),
                dict(tokens=4097), dict(logp=8193), dict(entropy=12289), dict(ids=16386),
                dict(lp=20481)):
        assert call(**bad) == -1, bad
    for bad in (dict(logp=4096 + 12), dict(entropy=8192), dict(ids=12288 + 12),
                dict(lp=16384 + 76), dict(logp=(1 << 20) + 1000 * 4 * 4 - 4),
                dict(lp=(1 << 20) - 76), dict(ids=8192 - 76)):
        assert call(**bad) == -1, bad
        assert b"overlaps" in lib.hy3x_last_error()
    assert call(T=0, logits=None, tokens=None, logp=None) == 0  # nothing to do


# ---------------------------------------------------------------- the definition
def definition(l, tokens, top, lowest, highest):
    """logp, entropy, ids, top_logp in 64 bits, and E|d|, E d^2 of each row."""
    T, V = l.shape
    l = np.minimum(l.astype(np.float64), highest) + 0.0
    with np.errstate(invalid="ignore"):
        l = np.where(l > lowest, l, -np.inf)
    m = l.max(1, keepdims=True)
    none = np.isneginf(m)
    d = l - np.where(none, 0.0, m)
    e = np.exp(d)
    S = e.sum(1, keepdims=True)
    p = e / np.where(none, 1.0, S)
    dz = np.where(np.isneginf(d), 0.0, d)
    lse = np.log(np.where(none, 1.0, S))
    lp = d - lse
    entropy = (lse - (p * dz).sum(1, keepdims=True))[:, 0]
    mine = np.take_along_axis(lp, np.clip(tokens, 0, V - 1)[:, None], 1)[:, 0]
    logp = np.where((tokens >= 0) & (tokens < V), mine, 0.0)
    ids = np.argsort(-l, axis=1, kind="stable")[:, :top].astype(np.int32)
    best = np.take_along_axis(lp, ids, 1)
    return logp, np.where(none[:, 0], 0.0, entropy), ids, best, (p * -dz).sum(1), (p * dz * dz).sum(1)


class Call:
    def __init__(self, torch, l, tokens, top, entropy=True):
        T, V = l.shape
        f32 = dict(dtype=torch.float32, device="cuda")
        self.l, self.tokens, self.T, self.V, self.top = l, tokens, T, V, top
        self.logp = torch.full((T,), 7.0, **f32)
        self.entropy = torch.full((T,), 7.0, **f32) if entropy else None
        self.ids = torch.full((T, top), -7, dtype=torch.int32, device="cuda") if top else None
        self.best = torch.full((T, top), 7.0, **f32) if top else None
        room = H.logprobs_workspace(T, V, top)
        self.ws = torch.full((room,), 255, dtype=torch.uint8, device="cuda") if room else None

    def __call__(self, stream=None):
        H.logprobs(self.l, self.tokens, self.T, self.logp, entropy=self.entropy, top_ids=self.ids,
                   top_logp=self.best, workspace=self.ws, stream=stream)
        return self

    def outputs(self):
        return [o for o in (self.logp, self.entropy, self.ids, self.best) if o is not None]


def check(torch, call, n=None):
    lim = torch.finfo(call.l.dtype)
    tokens = call.tokens.cpu().numpy()
    want = definition(call.l.float().cpu().numpy(), tokens, call.top, lim.min, lim.max)
    logp, entropy, ids, best, d1, d2 = want
    n = call.V / 256 + 8
    off = (n + 2 * d1) * HALF

    def near(got, exact, tol, what):
        got = got.double().cpu().numpy()
        same = (got == exact) | (np.abs(got - exact) <= tol + 2 * HALF * np.abs(exact))
        assert same.all(), (what, np.argwhere(~same)[:5].tolist(), got[~same][:5], exact[~same][:5])
    with np.errstate(invalid="ignore"):
        near(call.logp, logp, off, "logp")
        if call.entropy is not None:
            near(call.entropy, entropy, (n * (1 + d1) + 2 * d1 + 3 * d2) * HALF, "entropy")
        if call.top:
            assert np.array_equal(call.ids.cpu().numpy(), ids), \
                np.argwhere(call.ids.cpu().numpy() != ids)[:5].tolist()
            near(call.best, best, off[:, None], "top_logp")


def logits(torch, T, V, kind, seed, pad=0, at=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    flat = (spread * torch.randn(T * (V + pad) + at, generator=g)).to(getattr(torch, NAMES[kind]))
    return flat.cuda()[at:].view(T, V + pad)[:, :V]


def given(torch, T, V, seed):
    g = torch.Generator().manual_seed(seed + 100)
    return torch.randint(0, V, (T,), generator=g, dtype=torch.int32).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 31, 33, 63, 65, 255, 257, 511, 513, 1000, 2049,
                               4095, 4097, 8200, 16385, 32003])
def test_vocabularies(torch, V, kind):
    for T in (1, 3):
        for top in sorted({0, 1, min(V, 5), min(V, 20), min(V, 32)}):
            check(torch, Call(torch, logits(torch, T, V, kind, V + top, pad=T - 1, at=T - 1),
                              given(torch, T, V, V), top)())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
@pytest.mark.parametrize("T", [1, 2, 4, 7, 16, 33, 64, 130, 257, 600, 1100])
def test_rows(torch, T, kind):
    for V, top in ((700, 3), (6001, 20), (20011, 0)):
        check(torch, Call(torch, logits(torch, T, V, kind, T, pad=3), given(torch, T, V, T), top,
                          entropy=T % 2 == 1)())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
@pytest.mark.parametrize("T,V", [(1, 100), (1, 30000), (40, 5000), (1100, 700)])
def test_negative_logits(torch, T, V, kind):
    l = logits(torch, T, V, kind, V) - 60.0
    check(torch, Call(torch, l, given(torch, T, V, 1), 12)())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
def test_the_head_s_vocabulary(torch, kind):
    for T in (1, 2, 9):
        check(torch, Call(torch, logits(torch, T, 120832, kind, T), given(torch, T, 120832, T), 32)())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
@pytest.mark.parametrize("T", [1, 5, 300])
@pytest.mark.parametrize("V", [40, 1500, 40000])
def test_ties_and_orders(torch, V, T, kind):
    """Rows of equal values, of few values, rising, falling; the best at either end."""
    t = getattr(torch, NAMES[kind])
    g = torch.Generator().manual_seed(V)
    rise = torch.linspace(-9, 9, V).repeat(T, 1)
    few = torch.randint(-3, 4, (T, V), generator=g).float()
    ends = torch.randn(T, V, generator=g)
    ends[:, 0] = ends[:, V - 1] = 11.0
    zeros = torch.zeros(T, V)
    zeros[:, 1::2] = -0.0
    for l in (rise, rise.flip(1), few, torch.full((T, V), 1.25), ends, zeros):
        call = Call(torch, l.to(t).cuda(), given(torch, T, V, 3), min(V, 20))()
        check(torch, call)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
@pytest.mark.parametrize("V,T", [(50, 9), (3000, 9), (50021, 9), (50021, 300)])
def test_masks(torch, V, T, kind):
    """NaN, -inf and the type's lowest are one mask; rows with few tokens left, with one, with
    none; given tokens that are masked, or none."""
    t = getattr(torch, NAMES[kind])
    l = logits(torch, T, V, kind, V).clone()
    g = torch.Generator().manual_seed(V)
    off = torch.rand(T, V, generator=g) < 0.9
    off[1] = True                    # nothing left
    off[2] = True
    off[2, V // 2] = False           # one
    off[3] = True
    off[3, -3:] = False              # three, at the end
    kinds = torch.tensor([float("nan"), float("-inf"), torch.finfo(t).min], dtype=torch.float64)
    value = kinds[torch.randint(0, 3, (T, V), generator=g)].to(t)
    off, value = off.cuda(), value.cuda()
    l[off] = value[off]
    l[5, ::2] = float("inf")         # counts as the largest finite value
    l[6] = float("inf")
    l[7, 0] = float("inf")
    l[7, 1] = torch.finfo(t).max
    tokens = given(torch, T, V, 1)
    tokens[:5] = torch.tensor([-1, 3, V // 2, 0, V], dtype=torch.int32)
    check(torch, Call(torch, l, tokens, 20)())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
def test_one_token_has_it_all(torch, kind):
    """Entropies near 0, of rows whose other tokens have 1e-3 to 1e-14 of the mass."""
    T, V = 12, 5000
    l = logits(torch, T, V, kind, 3, spread=0.1).clone()
    l[:, 77] = torch.linspace(14.0, 42.0, T).to(l.dtype).cuda()
    tokens = torch.full((T,), 77, dtype=torch.int32, device="cuda")
    call = Call(torch, l, tokens, 5)()
    check(torch, call)
    lim = torch.finfo(l.dtype)
    _, entropy, *_ = definition(l.float().cpu().numpy(), tokens.cpu().numpy(), 5, lim.min, lim.max)
    got = call.entropy.double().cpu().numpy()
    # relative too: the sum of positive terms keeps its own precision, but for log S, of
    # which a part below 2^-24 of the largest term may be lost (at most a 14th of it at d = 14)
    assert (np.abs(got / entropy - 1) < 0.1).all(), (got, entropy)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_large_logits(torch, kind):
    """Values and differences of every size up to the type's largest."""
    t = getattr(torch, NAMES[kind])
    l = logits(torch, 6, 3001, kind, 3).float()
    scale = torch.tensor([1e3, 1e10, 1e30, 1e38, 1e-30, 50.0], device="cuda")[:, None]
    l = (l.double() * scale.double()).clamp(-3e38, 3e38).to(t)
    call = Call(torch, l, l.float().argmax(1).int(), 20)()
    check(torch, call)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(1, 120832), (40, 9001), (600, 3001)])
def test_graph_and_streams(torch, T, V):
    """Captured and replayed with other inputs, eager work between; two graphs; and calls at
    once, each with a workspace of its own."""
    calls = [Call(torch, logits(torch, T, V, "f32", i).clone(), given(torch, T, V, i), 8)()
             for i in range(3)]
    torch.cuda.synchronize()
    for c in calls:
        if V < 20000:
            check(torch, c)
    want = [[o.clone() for o in c.outputs()] for c in calls]
    into = Call(torch, calls[0].l.clone(), calls[0].tokens.clone(), 8)
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        into(torch.cuda.current_stream().cuda_stream)
    for i in (1, 2, 0, 1):
        into.l.copy_(calls[i].l)
        into.tokens.copy_(calls[i].tokens)
        for o in into.outputs():
            o.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(into.outputs(), want[i]))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, st in zip(calls, streams):
            c(st.cuda_stream)
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(c.outputs(), w))


@pytest.mark.gpu
def test_far_rows(torch):
    """Rows whose elements lie past 32-bit offsets."""
    far = (1 << 31) + 8
    room = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device="cuda")
    l = torch.as_strided(room, (3, 3000), (far, 1))
    l.copy_(torch.randn(3, 3000, generator=torch.Generator().manual_seed(2)))
    check(torch, Call(torch, l, given(torch, 3, 3000, 1), 5)())


@pytest.mark.gpu
def test_a_missing_workspace_is_refused(torch):
    l = logits(torch, 1, 120832, "f32", 1)
    call = Call(torch, l, given(torch, 1, 120832, 1), 4)
    room = H.logprobs_workspace(1, 120832, 4)
    if room:
        call.ws = None
        with pytest.raises(H.HY3XError, match="workspace"):
            call()
        call.ws = torch.empty(room - 1, dtype=torch.uint8, device="cuda")
        with pytest.raises(H.HY3XError, match="workspace"):
            call()


@pytest.mark.gpu
def test_head_then_logprobs(torch):
    """A run as they are used: hidden states, the head's logits, the token's probability and
    its alternatives; the rows of the logits lie in a wider buffer."""
    T, D, V = 5, 512, 7001
    g = torch.Generator().manual_seed(4)
    q = torch.randint(0, 16, (V, D), generator=g, dtype=torch.uint8)
    s = (0.02 * torch.rand(V, D // 128, generator=g)).bfloat16()
    head = H.Linear4(V, D, group=128, dtype="bf16")
    head.set((q[:, 0::2] | q[:, 1::2] << 4).contiguous().cuda(), s.cuda(), on_device=True)
    x = torch.randn(T, D, generator=g).cuda()
    buf = torch.full((T, V + 7), float("nan"), device="cuda")
    l = buf[:, :V]
    head.apply(x, l, T)
    exact = x.double().cpu() @ ((q.double() - 8) * s.double().repeat_interleave(128, 1)).t()
    assert (l.double().cpu() - exact).abs().max() < 1e-4
    check(torch, Call(torch, l, given(torch, T, V, 1), 20)())
    assert buf[:, V:].isnan().all()
    head.close()


@pytest.mark.gpu
def test_projection_with_adapters(torch):
    """y = W x in four bits, then the adapters of each token beside it, in place."""
    T, D, N, R = 9, 256, 300, 8
    g = torch.Generator().manual_seed(4)
    q = torch.randint(0, 16, (N, D), generator=g, dtype=torch.uint8)
    s = (0.02 * torch.rand(N, D // 64, generator=g)).bfloat16()
    proj = H.Linear4(N, D, group=64, dtype="bf16")
    proj.set((q[:, 0::2] | q[:, 1::2] << 4).contiguous().cuda(), s.cuda(), on_device=True)
    ad = H.Adapters(3, R, D, N, dtype="bf16")
    a, b = torch.randn(3, R, D, generator=g).bfloat16(), torch.randn(3, N, R, generator=g).bfloat16()
    for i in range(3):
        ad.set(i, a[i].cuda(), b[i].cuda(), scale=0.5, on_device=True)
    ids = torch.tensor([0, 1, 2, -1, 0, 1, 2, -1, 0], dtype=torch.int32)
    x = torch.randn(T, D, generator=g).cuda()
    y = torch.empty(T, N, device="cuda")
    proj.apply(x, y, T)
    ad.apply(ids.cuda(), x, y, T, base=y)
    xd = x.double().cpu()
    want = xd @ ((q.double() - 8) * s.double().repeat_interleave(64, 1)).t()
    for t in range(T):
        if ids[t] >= 0:
            want[t] += 0.5 * (b[ids[t]].double() @ (a[ids[t]].double() @ xd[t]))
    assert (y.double().cpu() - want).abs().max() < 1e-5 * want.abs().max()
    proj.close()
    ad.close()


@pytest.mark.gpu
def test_most_rows(torch):
    """More rows than a launch has threads for."""
    T, V = 1 << 24, 3
    g = torch.Generator(device="cuda").manual_seed(4)
    l = torch.randn(T, V, generator=g, device="cuda")
    tokens = torch.randint(0, V, (T,), generator=g, dtype=torch.int32, device="cuda")
    call = Call(torch, l, tokens, 2)()
    lp = torch.log_softmax(l.double(), 1)
    d = (lp.exp() * (l.double().amax(1, keepdim=True) - l)).sum(1)
    tol = (V / 256 + 8 + 2 * d) * HALF  # as in check
    mine = lp.gather(1, tokens.long()[:, None])[:, 0]
    assert ((call.logp - mine).abs() <= tol + 2 * HALF * mine.abs()).all()
    order = torch.sort(-l, dim=1, stable=True).indices[:, :2]
    assert torch.equal(call.ids.long(), order)
    best = lp.gather(1, order)
    assert ((call.best - best).abs() <= tol[:, None] + 2 * HALF * best.abs()).all()
    assert (call.entropy + (lp.exp() * lp).sum(1)).abs().max() < 1e-5
