"""The layer with a routing rule of its own and with adapters: routing, adapters
and experts in one forward, against the block's definition in 64 bits on the
layer's own weights. Outputs are held to the block's bar, relative L2 <= 1e-3 of
y - x (its experts work in fp16)."""
import ctypes

import numpy as np
import pytest

import hy3_amd as H
from hy3_amd import configs as C
from hy3_amd import hipmem
from oracle import hy3_oracle as O
from test_route_experts import oracle as route_oracle

D, F, E, TOL = 4096, 1536, 192, 1e-3
F32 = np.finfo(np.float32)


def test_null_refusals():
    lib, spec = H.lib(), H.RouteSpec()
    assert lib.hy3x_layer_set_routing(None, ctypes.byref(spec)) == -1
    assert lib.hy3x_layer_set_adapters(None, 0, None) == -1
    assert lib.hy3x_layer_forward_adapters(None, 4096, None, 4096, 1, 8, 2.826, None) == -1


# ---------------------------------------------------------------- on the GPU
@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


class Block:
    """A layer, its oracle (weights copied back from the device) and adapters of
    every projection whose products are as large as the projections' own."""

    COUNT = 3

    def __init__(self, torch, shared_q8=False):
        self.torch = torch
        self.layer = H.MoELayer(1500)
        self.layer.synth_experts(C.WEIGHT_SEED, 0)
        self.layer.set_router(*C.layer_small_tensors(C.WEIGHT_SEED))
        self.cpu = O.SynthLayer(C.WEIGHT_SEED, shared_q8=shared_q8)
        if shared_q8:
            self.layer.synth_shared_q8_0(C.WEIGHT_SEED, 0)
        self.shared_q8 = shared_q8
        self.mats = {}
        g = torch.Generator().manual_seed(11)
        shapes = {"router": (D, E), "gate": (D, F), "up": (D, F), "down": (F, D)}
        self.ab, self.handles = {}, {}
        for i, (p, (din, dout)) in enumerate(shapes.items()):
            dt, rank = ((torch.bfloat16, 8), (torch.float16, 16), (torch.bfloat16, 33),
                        (torch.float16, 5))[i]
            a = (torch.randn(self.COUNT, rank, din, generator=g) * 0.02).to(dt)
            b = (torch.randn(self.COUNT, dout, rank, generator=g) / rank ** 0.5).to(dt)
            h = H.Adapters(self.COUNT, rank, din, dout, "bf16" if dt == torch.bfloat16 else "f16")
            for k in range(self.COUNT):
                h.set(k, a[k].cuda(), b[k].cuda(), 1.0 + 0.25 * k, on_device=True)
            self.ab[p], self.handles[p] = (a.double().numpy(), b.double().numpy()), h

    def close(self):
        self.layer.close()
        for h in self.handles.values():
            h.close()

    def expert(self, e):
        """gate, up, down of expert e in 64 bits."""
        if e not in self.mats:
            if e == E and self.shared_q8:
                raw = self.cpu.expert(E)
                m = [O.dequant_q8(q) for q in raw]
            else:
                m = [O.dequant(hipmem.to_host(self.layer.expert_ptr(e, i), H.Q4K_MATRIX_BYTES))
                     for i in range(3)]
            self.mats[e] = tuple(v.astype(np.float64).reshape(s) for v, s in
                                 zip(m, ((F, D), (F, D), (D, F))))
        return self.mats[e]

    def delta(self, p, i, v):
        a, b = self.ab[p]
        return (1.0 + 0.25 * i) * (b[i] @ (a[i] @ v))

    def logits(self, x, ids, used):
        r = self.cpu.route(x)
        lg = r["logits"].astype(np.float64)
        for t, i in enumerate(ids):
            if "router" in used and 0 <= i < self.COUNT:
                lg[t] += self.delta("router", i, r["s"][t].astype(np.float64))
        return r["s"].astype(np.float64), lg

    def expect(self, x, s, adapter, chosen, w, used):
        """y - x of each token, its experts and weights given."""
        out = np.zeros((len(x), D))
        silu = lambda v: v / (1.0 + np.exp(-v))  # noqa: E731
        for t in range(len(x)):
            for e, we in zip(chosen[t], w[t]):
                g, u, d = self.expert(int(e))
                out[t] += we * (d @ (silu(g @ s[t]) * (u @ s[t])))
            g, u, d = self.expert(E)
            i = adapter[t]
            on = 0 <= i < self.COUNT
            gate, up = g @ s[t], u @ s[t]
            if on and "gate" in used:
                gate = gate + self.delta("gate", i, s[t])
            if on and "up" in used:
                up = up + self.delta("up", i, s[t])
            h = silu(gate) * up
            out[t] += d @ h
            if on and "down" in used:
                out[t] += self.delta("down", i, h)
        return out

    def use(self, used):
        for p in H.MoELayer.PROJECTIONS:
            self.layer.set_adapters(p, self.handles[p] if p in used else None)

    def run(self, x, adapter=None, K=8, attn=None, stream=None):
        torch, T = self.torch, len(x)
        xd = torch.from_numpy(np.ascontiguousarray(x, np.float32).copy()).cuda()
        ad = None if attn is None else torch.from_numpy(attn.copy()).cuda()
        if adapter is None:
            self.layer.forward(xd.data_ptr(), T, K)
        else:
            idd = torch.tensor(adapter, dtype=torch.int32).cuda()
            torch.cuda.synchronize()
            self.layer.forward_adapters(xd.data_ptr(), idd, T, K=K, stream=stream,
                                        attn_dev_ptr=None if ad is None else ad.data_ptr())
        torch.cuda.synchronize()
        ids, wpre, w = self.layer.last_routing(T, K)
        return xd.cpu().numpy(), ids, wpre, w


@pytest.fixture(scope="module", params=[False, True], ids=["q4k", "q8"])
def block(request, torch):
    b = Block(torch, request.param)
    yield b
    b.close()


@pytest.fixture(autouse=True)
def clean(request):
    yield
    if "block" in request.fixturenames:
        b = request.getfixturevalue("block")
        b.use(())
        b.layer.set_routing(None)
        b.layer.set_path(0)


def near_choice(ids, key, K):
    """Every choice is one that keys within 1e-5 allow (the adapted logits are fp32)."""
    for t in range(len(ids)):
        order = np.sort(key[t])[::-1][:K]
        assert len(set(ids[t])) == K
        assert (np.abs(key[t][ids[t]] - order) <= 1e-5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 40, 400])
def test_the_published_rule_as_a_rule(block, T):
    x = C.inputs(0xA0, T)
    block.layer.set_path(2)  # the MFMA tiles for one token too
    y0, ids0, wpre0, w0 = block.run(x)
    block.layer.set_routing(H.RouteSpec(E, 1, "sigmoid"))
    y, ids, wpre, w = block.run(x)
    assert np.array_equal(ids, ids0)
    assert (np.abs(wpre - wpre0) <= 60 * 2.0 ** -24 * wpre0).all()
    assert np.array_equal(w, wpre * np.float32(H.ROUTE_SCALE))
    # the experts' products are the same: what differs is the weights' last bits
    assert O.rel_l2(y - x, y0 - x) <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,spec", [
    (1, 8, dict(score="softmax")), (7, 8, dict(n_group=8, topk_group=4, group_score="top2")),
    (33, 3, dict(score="softmax", n_group=12, topk_group=5, renorm=False)),
    (64, 1, dict(n_group=64, topk_group=64)), (400, 8, dict(n_group=4, topk_group=1))])
def test_routing_rules(block, T, K, spec):
    x = C.inputs(0xA1, T)
    rule = H.RouteSpec(E, 1, **spec)
    block.layer.set_routing(rule)
    y, ids, wpre, w = block.run(x, K=K)
    s, lg = block.logits(x, [-1] * T, ())
    full = H.RouteSpec(E, K, **dict(spec, scale=1.0))
    want, ww, _ = route_oracle(full, lg.astype(np.float32), block.cpu.bias, F32.min, F32.max)
    assert np.array_equal(ids, want)
    assert (np.abs(wpre - ww) <= 80 * 2.0 ** -24 * ww).all()
    few = slice(0, 6)
    out = block.expect(x[few], s[few], [-1] * T, ids[few], w[few].astype(np.float64), ())
    assert O.rel_l2(y[few] - x[few], out) <= TOL


@pytest.mark.gpu
@pytest.mark.parametrize("used", [("router",), ("gate",), ("up",), ("down",),
                                  ("router", "gate", "up", "down")])
@pytest.mark.parametrize("T", [1, 2, 9])
def test_adapters(block, T, used):
    x = C.inputs(0xA2, T)
    adapter = [(0, 1, -1, 2, 3, 0, 2, -7, 1)[t] for t in range(T)]
    block.use(used)
    y, ids, wpre, w = block.run(x, adapter, K=4)
    s, lg = block.logits(x, adapter, used)
    sig = 1.0 / (1.0 + np.exp(-lg))
    near_choice(ids, sig + block.cpu.bias.astype(np.float64), 4)
    want = np.take_along_axis(sig, ids, 1)
    want = want / (want.sum(1, keepdims=True) + 1e-20)
    # adapted logits: fp32 sums over 4096 and 8, about 2e-5 of a logit of this size
    assert (np.abs(wpre - want) <= 2e-5).all()
    out = block.expect(x, s, adapter, ids, w.astype(np.float64), used)
    for t in range(T):
        assert O.rel_l2(y[t] - x[t], out[t]) <= TOL
    plain = block.expect(x, s, [-1] * T, ids, w.astype(np.float64), ())
    for t, i in enumerate(adapter):  # the adapters matter, or the test would not see them
        if used != ("router",) and 0 <= i < block.COUNT:
            assert O.rel_l2(plain[t], out[t]) > 0.05


@pytest.mark.gpu
@pytest.mark.parametrize("T", [30, 400, 1300])
def test_adapters_of_a_long_batch(block, T):
    """Each token as in a batch of few: the same experts, the result to the block's bar."""
    x = C.inputs(0xA3, T)
    adapter = [(t * 7 // 20) % 5 - 1 for t in range(T)]
    block.use(("router", "gate", "up", "down"))
    block.layer.set_routing(H.RouteSpec(E, 1, "sigmoid", 8, 4, "top2"))
    y, ids, _, w = block.run(x, adapter)
    for at in range(0, T, max(1, T // 6)):
        part = slice(at, min(at + 3, T))
        yp, idp, _, wp = block.run(x[part], adapter[part])
        if np.array_equal(idp, ids[part]):  # near ties of adapted logits may differ
            assert O.rel_l2(y[part] - x[part], yp - x[part]) <= TOL / 2
        else:
            assert (np.sort(idp) != np.sort(ids[part])).sum() <= 2


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 5, 40, 400, 1300])
def test_without_an_adapter_the_block_is_as_it_was(block, T):
    x = C.inputs(0xA4, T)
    y0, ids0, wpre0, w0 = block.run(x)
    block.use(("router", "gate", "up", "down"))
    y, ids, wpre, w = block.run(x, [-1, 3][T % 2:] * T if T < 3 else [-1] * T)
    assert np.array_equal(ids, ids0) and np.array_equal(wpre, wpre0) and np.array_equal(w, w0)
    # other tile shapes above 1152 tokens are the same arithmetic
    assert np.array_equal(y, y0)
    y1, ids1, _, _ = block.run(x)  # and forward uses none of them
    assert np.array_equal(y1, y0) and np.array_equal(ids1, ids0)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6])
def test_no_adapters_set(block, T):
    x = C.inputs(0xAA, T)
    y0, ids0, _, _ = block.run(x)
    y, ids, _, _ = block.run(x, [0] * T)  # ids name adapters of no projection
    assert np.array_equal(y, y0) and np.array_equal(ids, ids0)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 9, 64])
def test_rule_on_the_static_scratch_and_the_gemv_path(block, T):
    torch, layer = block.torch, block.layer
    x = C.inputs(0xAB, T)
    layer.set_routing(H.RouteSpec(E, 1, "softmax", 4, 2, "top2"))
    y0, ids0, wpre0, _ = block.run(x)
    xd = torch.from_numpy(x.copy()).cuda()
    layer.forward_static(xd.data_ptr(), T)
    torch.cuda.synchronize()
    ids, wpre, _ = layer.last_routing()
    assert np.array_equal(xd.cpu().numpy(), y0)
    assert np.array_equal(ids, ids0) and np.array_equal(wpre, wpre0)
    if not block.shared_q8:
        layer.set_path(1)
        y1, ids1, wpre1, _ = block.run(x)
        assert np.array_equal(ids1, ids0) and np.array_equal(wpre1, wpre0)
        assert O.rel_l2(y1 - x, y0 - x) <= TOL


@pytest.mark.gpu
def test_residual_and_two_layers_with_one_scratch(torch):
    b = Block(torch)
    other = H.MoELayer(0, share_scratch_with=b.layer)
    try:
        T = 11
        x, attn = C.inputs(0xA5, T), C.inputs(0xA6, T)
        adapter = [t % 4 - 1 for t in range(T)]
        b.use(("gate", "down"))
        want, ids, _, _ = b.run(x + attn, adapter)
        got, ids2, _, _ = b.run(x, adapter, attn=attn)
        assert np.array_equal(ids, ids2) and np.array_equal(got, want)
        # the same weights, the other handle of the same scratch
        for e in range(E + 1):
            other.set_expert_q4k(e, *(b.layer.expert_ptr(e, m) for m in range(3)), on_device=True)
        other.set_router(*C.layer_small_tensors(C.WEIGHT_SEED))
        other.set_adapters("gate", b.handles["gate"])
        other.set_adapters("down", b.handles["down"])
        xd = torch.from_numpy((x + attn).copy()).cuda()
        idd = torch.tensor(adapter, dtype=torch.int32).cuda()
        other.forward_adapters(xd.data_ptr(), idd, T)
        torch.cuda.synchronize()
        assert np.array_equal(xd.cpu().numpy(), want)
        with pytest.raises(H.HY3XError):
            b.layer.last_routing()
    finally:
        other.close()
        b.close()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6, 500])
def test_graph_replays(block, T):
    torch = block.torch
    block.use(("router", "gate", "up", "down"))
    block.layer.set_routing(H.RouteSpec(E, 1, "softmax", 8, 4, "max"))
    sets = [(C.inputs(0xA7 + i, T), [(t + i) % 4 - 1 for t in range(T)]) for i in range(2)]
    want = [block.run(x, a)[0] for x, a in sets]
    xd = torch.zeros(T, D, device="cuda")
    idd = torch.zeros(T, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.layer.forward_adapters(xd.data_ptr(), idd, T,
                                     stream=torch.cuda.current_stream().cuda_stream)
    for i in (0, 1, 1, 0):
        xd.copy_(torch.from_numpy(sets[i][0]))
        idd.copy_(torch.tensor(sets[i][1], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(xd.cpu().numpy(), want[i])
        assert np.array_equal(block.run(*sets[1 - i])[0], want[1 - i])  # eager between replays


@pytest.mark.gpu
def test_refusals(block):
    torch, layer = block.torch, block.layer
    with pytest.raises(H.HY3XError, match="n_expert"):
        layer.set_routing(H.RouteSpec(128, 8))
    with pytest.raises(H.HY3XError, match="n_group"):
        layer.set_routing(H.RouteSpec(E, 8, n_group=5))
    with pytest.raises(H.HY3XError, match="projection"):
        layer.set_adapters("gate", block.handles["down"])
    lib = H.lib()
    assert lib.hy3x_layer_set_adapters(layer._h, 4, None) == -1
    assert lib.hy3x_layer_set_adapters(layer._h, -1, None) == -1
    x = torch.zeros(4, D, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    call = lambda a, i, T=4, K=8: lib.hy3x_layer_forward_adapters(  # noqa: E731
        layer._h, x.data_ptr(), a, i, T, K, 2.826, None)
    assert call(None, None) == -1 and call(None, ids.data_ptr() + 1) == -1
    assert call(x.data_ptr(), ids.data_ptr()) == -1 and b"overlaps" in lib.hy3x_last_error()
    assert call(None, ids.data_ptr(), T=0) == -1 and call(None, ids.data_ptr(), K=9) == -1
    layer.set_routing(H.RouteSpec(E, 1, n_group=32, topk_group=1))
    with pytest.raises(H.HY3XError, match="kept groups"):
        layer.forward(x.data_ptr(), 4, 7)
    layer.forward(x.data_ptr(), 4, 6)
    layer.set_routing(None)
    block.use(("gate",))
    if not block.shared_q8:
        layer.set_path(1)
        with pytest.raises(H.HY3XError, match="GEMV"):
            layer.forward_adapters(x.data_ptr(), ids, 4)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_ids_on_x_and_closed_adapters_are_refused(block):
    torch, layer = block.torch, block.layer
    x = torch.zeros(4, D, device="cuda")
    for at in (x.data_ptr(), x.data_ptr() - 12, x.data_ptr() + 4 * (4 * D - 1)):
        with pytest.raises(H.HY3XError, match="adapter_ids overlaps x"):
            layer.forward_adapters(x.data_ptr(), at, 4)
    with pytest.raises(TypeError):
        layer.forward_adapters(x.data_ptr(), np.zeros(4, np.int32), 4)
    h = H.Adapters(1, 8, D, E, "f16")
    h.close()
    with pytest.raises(H.HY3XError, match="closed"):
        layer.set_adapters("router", h)


@pytest.mark.gpu
def test_kernel_names_and_replays(block):
    torch, layer = block.torch, block.layer
    block.use(("gate",))
    x = torch.from_numpy(C.inputs(0xA9, 400).copy()).cuda()
    ids = torch.zeros(400, dtype=torch.int32, device="cuda")
    for T, name in ((4, "mfma_raw::"), (400, "mfma_raw_wide::")):
        layer.forward_adapters(x.data_ptr(), ids, T)
        assert layer.last_kernel("gateup").startswith(name)
        for stage in H.MoELayer.STAGES:
            assert layer.time_stage(stage, 2) >= 0.0
    layer.forward(x.data_ptr(), 400)
    assert layer.last_kernel("gateup").startswith("mfma_wide::")


@pytest.mark.gpu
def test_adapters_closed_while_set_are_refused(block):
    torch, layer = block.torch, block.layer
    x = torch.from_numpy(C.inputs(0xAC, 6).copy()).cuda()
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    h = H.Adapters(1, 8, D, F, "f16")
    layer.set_adapters("up", h)
    layer.forward_adapters(x.data_ptr(), ids, 6)
    torch.cuda.synchronize()
    h.close()
    with pytest.raises(H.HY3XError, match="closed"):
        layer.forward_adapters(x.data_ptr(), ids, 6)
    with pytest.raises(H.HY3XError, match="closed"):
        layer.time_stage("gateup", 1)
    layer.set_adapters("up", None)
    layer.forward_adapters(x.data_ptr(), ids, 6)  # none set: the block as it is
    assert layer.time_stage("gateup", 1) >= 0.0
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [30, 400, 1300])
@pytest.mark.parametrize("runs", [1, 20])
def test_a_long_batch_against_the_definition(block, T, runs):
    """Tokens from all over a batch in adapter tiles of 16 and in the wide expert tiles,
    each with an adapter of its own or in requests: the experts are ones that the 64-bit
    keys allow, and the outputs those of the definition for these experts and weights."""
    x = C.inputs(0xAD, T)
    adapter = [(t * 7 // runs) % 5 - 1 for t in range(T)]
    used = ("router", "gate", "up", "down")
    block.use(used)
    y, ids, wpre, w = block.run(x, adapter)
    at = sorted({0, 1, T // 3, T // 2, T - 17, T - 1})  # first and last tiles, tails
    ad = [adapter[t] for t in at]
    s, lg = block.logits(x[at], ad, used)
    sig = 1.0 / (1.0 + np.exp(-lg))
    near_choice(ids[at], sig + block.cpu.bias.astype(np.float64), 8)
    want = np.take_along_axis(sig, ids[at], 1)
    want = want / (want.sum(1, keepdims=True) + 1e-20)
    assert (np.abs(wpre[at] - want) <= 2e-5).all()
    out = block.expect(x[at], s, ad, ids[at], w[at].astype(np.float64), used)
    for i, t in enumerate(at):
        assert O.rel_l2(y[t] - x[t], out[i]) <= TOL
