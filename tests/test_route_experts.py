"""hy3x_route_experts against the definition in 64 bits (numpy, row by row).

Indices have to be equal. The weights' tolerance counts the roundings of an
fp32 evaluation (2^-24 each, half a step): the exponential's argument
(|l - max| of them, as exp turns an absolute error into a relative one), exp
(2 ulp = 4), the sum over up to 1024 experts in a wave (16 + 6), the sum and
division of the renormalisation over up to 16 (16 + 2), the scale (1)."""
import ctypes

import numpy as np
import pytest

import hy3_amd as H

HALF = 2.0 ** -24


def oracle(spec, logits, bias, lowest, highest):
    """ids, w and the largest |l - max| of a chosen expert of each row."""
    T, E = logits.shape
    size = E // spec.n_group
    softmax, top2 = spec.score == 1, spec.group_score == 1
    ids = np.empty((T, spec.k), np.int32)
    w = np.zeros((T, spec.k))
    reach = np.zeros(T)
    for t in range(T):
        l = np.minimum(logits[t].astype(np.float64), highest)
        on = l > lowest
        if bias is not None:
            on &= bias > -np.inf
        s = np.zeros(E)
        if not softmax:
            s[on] = 1.0 / (1.0 + np.exp(-l[on]))
        elif on.any():
            e = np.exp(l[on] - l[on].max())
            s[on] = e / e.sum()
        scored = s if bias is None else s + bias.astype(np.float64)
        key = l if bias is None else scored
        groups = []
        for g in range(spec.n_group):
            part = slice(g * size, (g + 1) * size)
            v = np.sort((scored if top2 else key)[part][on[part]])[::-1]
            groups.append((v.size == 0, -(v[:2].sum() if top2 else v[0]) if v.size else 0.0, g))
        kept = {g for _, _, g in sorted(groups)[:spec.topk_group]}
        place = [(e // size not in kept, not on[e], -key[e] if on[e] else 0.0, e)
                 for e in range(E)]
        ids[t] = [p[3] for p in sorted(place)[:spec.k]]
        v = s[ids[t]]
        if spec.renorm:
            v = v / (v.sum() + 1e-20)
        w[t] = v * np.float64(np.float32(spec.scale))
        live = ids[t][on[ids[t]]]
        if live.size:
            reach[t] = np.abs(l[live] - (l[on].max() if softmax else 0.0)).max()
    return ids, w, reach


# ---------------------------------------------------------------- refusals (no GPU)
GOOD = dict(n_expert=192, k=8, n_group=8, topk_group=4)


@pytest.mark.parametrize("change,word", [
    (dict(n_expert=0), "n_expert"), (dict(n_expert=1025), "n_expert"), (dict(k=0), "k 0"),
    (dict(k=17), "k 17"), (dict(n_group=0), "n_group"), (dict(n_group=7), "divisor"),
    (dict(n_group=96), "n_group"), (dict(topk_group=0), "topk_group"),
    (dict(topk_group=9), "topk_group"), (dict(n_expert=8, k=5), "kept groups")])
def test_spec_refusals(change, word):
    spec = H.RouteSpec(**dict(GOOD, **change))
    with pytest.raises(H.HY3XError, match=word):
        H.route_experts(spec, 4096, 1, 4096, 4096)


def test_host_memory_refusals():
    import torch
    spec = H.RouteSpec(**GOOD)
    logits, ids, w = torch.zeros(1, 192), torch.zeros(1, 8, dtype=torch.int32), torch.zeros(1, 8)
    for args in ((logits, 1, 4096, 4096), (4096, 1, ids, 4096), (4096, 1, 4096, w),
                 (logits.numpy(), 1, 4096, 4096), (4096, 1, ids.numpy(), 4096)):
        with pytest.raises(TypeError):
            H.route_experts(spec, *args)
    with pytest.raises(TypeError):
        H.route_experts(spec, 4096, 1, 4096, 4096, bias=w)


def test_argument_refusals():
    lib, spec = H.lib(), H.RouteSpec(**GOOD)

    def call(spec=spec, logits=4096, dtype=0, stride=192, bias=None, T=1, ids=4096, w=4096):
        return lib.hy3x_route_experts(ctypes.byref(spec) if spec else None, logits, dtype, stride,
                                      bias, T, ids, w, None)
    assert call(spec=None) == -1
    assert call(dtype=3) == -1 and call(dtype=-1) == -1
    assert call(stride=191) == -1 and call(stride=(1 << 32) + 1) == -1
    assert call(T=-1) == -1 and call(T=(1 << 24) + 1) == -1
    assert call(logits=None) == -1 and call(ids=None) == -1 and call(w=None) == -1
    assert call(logits=4098) == -1 and call(bias=4097) == -1
    assert call(ids=4097) == -1 and call(w=4098) == -1
    assert b"aligned" in lib.hy3x_last_error()
    far = dict(ids=1 << 20, w=2 << 20)  # 8 x 4 bytes each
    for bad in (dict(w=(1 << 20) + 28), dict(ids=4096 + 188 * 4), dict(w=4096), dict(logits=(2 << 20) + 4),
                dict(bias=(1 << 20) - 4), dict(T=3, ids=4096 + 2 * 192 * 4)):
        assert call(**dict(far, **bad)) == -1, bad
        assert b"overlaps" in lib.hy3x_last_error()
    for field in ("score", "group_score"):
        bad = H.RouteSpec(**GOOD)
        setattr(bad, field, 2)
        assert call(spec=bad) == -1
    assert call(T=0, logits=None, ids=None, w=None) == 0  # nothing to do


# ---------------------------------------------------------------- on the GPU
@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


def make(torch, T, E, dtype, seed, spread=1.28):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(T, E, generator=g)).to(
        {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])


def run(torch, spec, logits, dtype, bias=None, pad=0, stream=None):
    """Device call on a copy of `logits`, rows `pad` elements apart; a guard behind
    the outputs stays as it was."""
    T, E = logits.shape
    wide = torch.full((T, E + pad), 7.0, dtype=logits.dtype)
    wide[:, :E] = logits
    lg = wide.cuda()
    b = None if bias is None else torch.from_numpy(bias).cuda()
    ids = torch.full((T * spec.k + 5,), -77, dtype=torch.int32, device="cuda")
    w = torch.full((T * spec.k + 5,), -7.0, device="cuda")
    torch.cuda.synchronize()
    H.route_experts(spec, lg, T, ids, w, dtype=dtype, row_stride=E + pad, bias=b, stream=stream)
    torch.cuda.synchronize()
    ids, w = ids.cpu().numpy(), w.cpu().numpy()
    n = T * spec.k
    assert (ids[n:] == -77).all() and (w[n:] == -7.0).all()
    return ids[:n].reshape(T, -1), w[:n].reshape(T, -1)


def check(torch, spec, logits, dtype, bias=None, pad=0):
    info = torch.finfo(logits.dtype)
    want, w, reach = oracle(spec, logits.float().numpy(), bias, info.min, info.max)
    ids, got = run(torch, spec, logits, dtype, bias, pad)
    assert np.array_equal(ids, want)
    tol = (45 + reach[:, None]) * HALF * np.abs(w) + 2.0 ** -149 * abs(spec.scale)
    assert (np.abs(got - w) <= tol).all()


def bias_of(E, seed, span=0.1):
    return np.random.default_rng(seed).uniform(-span, span, E).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,k,groups,kept", [
    (1, 1, 1, 1, 1), (1, 192, 8, 1, 1), (3, 61, 7, 1, 1), (17, 64, 16, 1, 1), (5, 65, 8, 5, 2),
    (33, 192, 8, 8, 4), (7, 251, 6, 1, 1), (64, 256, 8, 8, 3), (9, 384, 8, 16, 4),
    (4, 1000, 10, 20, 5), (6, 1024, 16, 64, 64), (12, 64, 2, 64, 3), (130, 160, 1, 4, 1),
    (2, 513, 16, 3, 1)])
def test_route(torch, dtype, score, T, E, k, groups, kept):
    for i, (best, bias, renorm) in enumerate([("max", True, True), ("top2", True, False),
                                              ("max", False, False), ("top2", False, True)]):
        spec = H.RouteSpec(E, k, score, groups, kept, best, renorm, 2.826)
        check(torch, spec, make(torch, T, E, dtype, 100 * i + T), dtype,
              bias_of(E, i, 0.1 if score == "sigmoid" else 0.01) if bias else None,
              pad=(0, 3, 8, 1)[i])


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,groups", [(4097, 192, 1), (16383, 256, 8), (70001, 32, 4)])
def test_many_rows(torch, T, E, groups):
    """Every row against a plain sort on the device (the row-by-row oracle is slow)."""
    logits = make(torch, T, E, "f32", 5).cuda()
    bias = torch.from_numpy(bias_of(E, 6)).cuda()
    spec = H.RouteSpec(E, 8, "sigmoid", groups, max(1, groups // 2), "max", True, 1.0)
    ids = torch.empty(T, 8, dtype=torch.int32, device="cuda")
    w = torch.empty(T, 8, device="cuda")
    H.route_experts(spec, logits, T, ids, w, bias=bias)
    s = 1.0 / (1.0 + torch.exp(-logits.double()))
    key = s + bias.double()
    if groups > 1:
        member = key.view(T, groups, -1)
        kept = torch.sort(member.amax(2), dim=1, descending=True, stable=True).indices[:, :groups // 2]
        stays = torch.zeros(T, groups, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        key = torch.where(stays[:, :, None], member, -9.0).view(T, E)
    want = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(ids, want.int())
    v = s.gather(1, want)
    v = v / v.sum(1, keepdim=True)
    assert ((w - v).abs() <= 60 * HALF * v).all()


def special_rows(E, dtype, torch):
    """Rows with ties, masks, infinities and NaN in every place that matters."""
    kind = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    info = torch.finfo(kind)
    inf, nan = float("inf"), float("nan")
    base = make(torch, 1, E, dtype, 3)[0].float()
    rows = [torch.zeros(E), torch.full((E,), 2.5), torch.full((E,), -inf), torch.full((E,), nan),
            torch.full((E,), info.min), torch.full((E,), info.max), torch.full((E,), inf)]
    for v in (-inf, nan, info.min, inf, info.max):
        for step in (2, E - 1):
            r = base.clone()
            r[::step] = v
            rows.append(r)
    one = torch.full((E,), -inf)
    one[E // 2] = 0.25
    rows.append(one)
    one = torch.full((E,), nan)
    one[E - 1] = -3.0
    rows.append(one)
    ties = base.round()
    rows += [ties, (2 * base).round() / 2, torch.full((E,), -200.0), base - 95.0, base - 60.0,
             base * 30.0]
    return torch.stack(rows).to(kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,groups,kept,best", [(64, 1, 1, "max"), (192, 8, 4, "top2"),
                                                (192, 8, 4, "max"), (63, 9, 3, "top2"),
                                                (256, 64, 5, "top2"), (10, 10, 7, "top2")])
def test_special_rows(torch, dtype, score, E, groups, kept, best):
    logits = special_rows(E, dtype, torch)
    k = min(7, kept * (E // groups))
    flat = np.zeros(E, np.float32)
    few = np.where(np.arange(E) % 3 == 0, 0.05, 0.0).astype(np.float32)
    odd = bias_of(E, 1)
    odd[0], odd[E // 3], odd[E - 1] = -np.inf, np.nan, np.inf
    # one ulp of fp32 apart: decided by the scores' low bits
    near = (0.5 + np.arange(E) * 2.0 ** -24).astype(np.float32)
    for bias in (None, flat, few, odd, near):
        for renorm in (True, False):
            check(torch, H.RouteSpec(E, k, score, groups, kept, best, renorm, 2.0), logits, dtype,
                  bias)


@pytest.mark.gpu
def test_keys_closer_than_fp32(torch):
    """s + bias equal in fp32 and different in 64 bits: the larger one first."""
    E = 64
    logits = torch.full((40, E), -4.0)
    g = torch.Generator().manual_seed(9)
    logits += torch.randint(-3, 4, (40, E), generator=g) * 2.0 ** -20
    bias = np.full(E, 0.75, np.float32)
    for score in ("sigmoid", "softmax"):
        for groups, best in ((1, "max"), (8, "max"), (8, "top2")):
            check(torch, H.RouteSpec(E, 8, score, groups, max(1, groups // 2), best), logits, "f32",
                  bias)


@pytest.mark.gpu
def test_rows_more_than_2_31_elements_apart(torch):
    E, stride, k = 192, (1 << 31) + 5, 8
    logits = make(torch, 2, E, "bf16", 4)
    buf = torch.empty(stride + E, dtype=torch.bfloat16, device="cuda")
    buf[:E], buf[stride:] = logits[0].cuda(), logits[1].cuda()
    ids = torch.empty(2, k, dtype=torch.int32, device="cuda")
    w = torch.empty(2, k, device="cuda")
    H.route_experts(H.RouteSpec(E, k), buf, 2, ids, w, dtype="bf16", row_stride=stride)
    torch.cuda.synchronize()
    want, _ = run(torch, H.RouteSpec(E, k), logits, "bf16")
    assert np.array_equal(ids.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_types_of_tensors(torch, dtype):
    spec = H.RouteSpec(192, 8)
    logits = make(torch, 5, 192, dtype, 3)
    want = run(torch, spec, logits, dtype)
    logits, bias = logits.cuda(), torch.zeros(192, dtype=torch.float64, device="cuda")
    ids = torch.zeros(5, 8, dtype=torch.int32, device="cuda")
    w = torch.zeros(5, 8, device="cuda")
    H.route_experts(spec, logits, 5, ids, w)  # the logits' own type
    torch.cuda.synchronize()
    assert np.array_equal(ids.cpu().numpy(), want[0])
    assert np.array_equal(w.cpu().numpy(), want[1])
    for bad in (dict(ids=ids.long()), dict(w=w.double()), dict(logits=logits.double()),
                dict(bias=bias)):
        with pytest.raises(TypeError):
            H.route_experts(spec, **dict(dict(logits=logits, T=5, ids=ids, w=w), **bad))


@pytest.mark.gpu
def test_streams_and_graph(torch):
    spec = H.RouteSpec(192, 8, "softmax", 8, 4, "top2")
    a, b = make(torch, 300, 192, "f32", 1), make(torch, 300, 192, "f32", 2)
    wa, wb = run(torch, spec, a, "f32"), run(torch, spec, b, "f32")
    lg = a.cuda()
    ids = [torch.zeros(300, 8, dtype=torch.int32, device="cuda") for _ in range(2)]
    w = [torch.zeros(300, 8, device="cuda") for _ in range(2)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    lb = b.cuda()
    torch.cuda.synchronize()
    H.route_experts(spec, lg, 300, ids[0], w[0], stream=s1.cuda_stream)  # two at once
    H.route_experts(spec, lb, 300, ids[1], w[1], stream=s2.cuda_stream)
    torch.cuda.synchronize()
    for i, want in enumerate((wa, wb)):
        assert np.array_equal(ids[i].cpu().numpy(), want[0])
        assert np.array_equal(w[i].cpu().numpy(), want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        H.route_experts(spec, lg, 300, ids[0], w[0],
                        stream=torch.cuda.current_stream().cuda_stream)
    for src, want in ((b, wb), (a, wa), (b, wb)):
        lg.copy_(src)
        ids[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(ids[0].cpu().numpy(), want[0])
        assert np.array_equal(w[0].cpu().numpy(), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("span", [12.0, 1e4, 1e6, 3e7])
@pytest.mark.parametrize("E,groups,kept", [(64, 32, 5), (192, 8, 4), (256, 16, 8), (1000, 20, 5)])
def test_sums_of_two_that_cancel(torch, score, span, E, groups, kept):
    """One expert of each group pinned by a large bias, the others held off by its
    negative: a group's score is what is left of the two, far below their rounding in
    fp32, and the groups still come in the order of 64 bits."""
    logits = make(torch, 60, E, "f32", 21)
    bias = np.full(E, -span, np.float32)
    bias[np.arange(groups) * (E // groups) + np.arange(groups) % (E // groups)] = span
    check(torch, H.RouteSpec(E, 5, score, groups, kept, "top2"), logits, "f32", bias)


# Lanes that hold 8 experts, and those that hold more and read their logits again:
# without groups 512 (8 a lane), 320 (5), 1024 (16); 1000 in 20 groups (25 of 32), 1024 in
# 64 groups (16), 360 in 3 (8).
WIDE = [(320, 1, 1), (512, 1, 1), (1024, 1, 1), (360, 3, 2), (1000, 20, 7), (1024, 64, 9)]


def check_wide(torch, spec, logits, dtype, bias=None, pad=0):
    """check() with the weights' tolerance for lanes of up to 32 experts: the argument
    (reach), exp (4), the softmax's sum of 32 a lane and 64 lanes (32 + 6) of terms off by
    (1.5 |x| + 4) roundings of themselves (at most 11 of the sum of 1024, as |x| exp(-|x|)
    falls), the renormalisation (18), the scale (1)."""
    info = torch.finfo(logits.dtype)
    want, w, reach = oracle(spec, logits.float().numpy(), bias, info.min, info.max)
    ids, got = run(torch, spec, logits, dtype, bias, pad)
    assert np.array_equal(ids, want)
    tol = (72 + reach[:, None]) * HALF * np.abs(w) + 2.0 ** -149 * abs(spec.scale)
    assert (np.abs(got - w) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,groups,kept", WIDE)
def test_rows_of_wide_lanes(torch, dtype, score, E, groups, kept):
    for i, (best, bias, renorm) in enumerate([("max", True, True), ("top2", True, False),
                                              ("max", False, False), ("top2", False, True)]):
        spec = H.RouteSpec(E, 16 - i, score, groups, kept, best, renorm, 2.5)
        check_wide(torch, spec, make(torch, 70, E, dtype, 10 * i + E), dtype,
                   bias_of(E, i, 0.1 if score == "sigmoid" else 0.01) if bias else None,
                   pad=(0, 3, 8, 1)[i])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("best", ["max", "top2"])
@pytest.mark.parametrize("E,groups,kept", WIDE)
def test_special_rows_of_wide_lanes(torch, dtype, score, best, E, groups, kept):
    logits = special_rows(E, dtype, torch)
    odd = bias_of(E, 1)
    odd[0], odd[E // 3], odd[E - 1] = -np.inf, np.nan, np.inf
    near = (0.5 + np.arange(E) * 2.0 ** -24).astype(np.float32)
    for bias in (None, np.zeros(E, np.float32), odd, near):
        for renorm in (True, False):
            spec = H.RouteSpec(E, 7, score, groups, kept, best, renorm, 2.0)
            check_wide(torch, spec, logits, dtype, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,groups,kept", WIDE + [(192, 1, 1), (256, 8, 4)])
def test_more_near_ties_than_lanes(torch, score, E, groups, kept):
    """Every expert within fp32's margin of every other: more candidates than a wave has
    lanes, all of them in the order of 64 bits."""
    g = torch.Generator().manual_seed(E)
    logits = -4.0 + torch.randint(-40, 41, (12, E), generator=g) * 2.0 ** -20
    bias = np.full(E, 0.75, np.float32)
    for best in ("max", "top2"):
        check_wide(torch, H.RouteSpec(E, 8, score, groups, kept, best), logits, "f32", bias)
