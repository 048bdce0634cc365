"""Routing to experts and low-rank adapters, as measurable cases.

Two operators that stand beside the MoE FFN block:

  route      hy3_amd.route_experts: scores of given router logits (sigmoid or
             softmax), a bias that steers the choice, groups of experts, top-k,
             renormalised weights;
  adapters   hy3_amd.Adapters: the low-rank adapters of many requests at once,
             y = base + scale_a * B_a (A_a x), beside a shared projection's
             output `base`.

Where `own` is false, run() computes them in their plain form: elementary torch
operations in 32 bits, the keys that choose experts in 64.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def route(name, tokens, experts, k, score="sigmoid", bias=True, groups=1, kept=1, best="max",
          renorm=True, scale=1.0, dtype="f32", masked=0.0):
    c = {"op": "route", "tokens": tokens, "experts": experts, "k": k, "score": score,
         "bias": bias, "groups": groups, "kept": kept, "best": best, "renorm": renorm,
         "scale": scale, "dtype": dtype, "masked": masked}
    return dict(c, name=name) if name else c


def adapters(name, tokens, d_in, d_out, rank, count, weights="bf16", io="same", mixed=False,
             run=1, pad=0):
    """mixed: each token has an adapter of its own choice; else requests of about
    `run` tokens, each with one adapter. pad: elements between the rows of x."""
    c = {"op": "adapters", "tokens": tokens, "d_in": d_in, "d_out": d_out, "rank": rank,
         "count": count, "weights": weights, "io": io, "mixed": mixed, "run": run, "pad": pad}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the decode step of one sequence: 192 experts, the published rule
        route("route_1", 1, 192, 8, scale=2.826),
        # a small decode batch, softmax scores in bf16 limited to half the groups
        route("route_32_softmax_groups", 32, 256, 6, score="softmax", bias=False, groups=8,
              kept=4, dtype="bf16"),
        # an ordinary prefill chunk, some experts pruned
        route("route_512_pruned", 512, 192, 8, scale=2.826, masked=0.1),
        # a long chunk, experts of at most four of eight devices per token
        route("route_4096_groups", 4096, 256, 8, groups=8, kept=4, best="top2", scale=2.5),
        # the largest: a whole batch's prefill, an odd expert count, no renormalisation
        route("route_16383_odd", 16383, 251, 7, score="softmax", bias=True, renorm=False,
              dtype="f16"),
        # one decoded token, beside the router (fp32 activations and logits)
        adapters("adapters_1_router", 1, 4096, 192, 8, 4, io="f32"),
        # a decode batch, almost every sequence with another adapter, beside the shared
        # expert's gate
        adapters("adapters_32_decode", 32, 4096, 1536, 16, 64, mixed=True),
        # odd everything: tokens, widths, rank, rows of a wider buffer
        adapters("adapters_61_odd", 61, 1001, 777, 5, 7, weights="f16", mixed=True, pad=3),
        # a large decode batch
        adapters("adapters_256_decode", 256, 4096, 4096, 16, 128, mixed=True),
        # a prefill chunk beside the shared expert's down projection, fp32 activations
        adapters("adapters_512_down_f32", 512, 1536, 4096, 32, 8, weights="f16", io="f32",
                 run=200),
        # ragged prompts of many requests
        adapters("adapters_2000", 2000, 4096, 4096, 16, 32, run=150),
        # the longest chunk, with adapters of a high rank
        adapters("adapters_4096_rank64", 4096, 4096, 4096, 64, 32, weights="f16", run=400),
    ]


def spread(rng, low, high):
    """A whole number in [low, high], even over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    if rng.random() < 0.45:
        tokens = spread(rng, 1, 16383)
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * spread(rng, 8, 512 // groups) if groups > 1 else spread(rng, 32, 512)
        if tokens * experts > 16383 * 251:
            tokens = 16383 * 251 // experts
        kept = rng.randint(1, groups)
        k = min(rng.choice([8, 8, 8, 7, 6, 4, 2, 1]), kept * (experts // groups))
        return route(None, tokens, experts, k, score=rng.choice(["sigmoid", "softmax"]),
                     bias=rng.random() < 0.6, groups=groups, kept=kept,
                     best=rng.choice(["max", "top2"]), renorm=rng.random() < 0.7,
                     scale=rng.choice([1.0, 2.5, 2.826]), dtype=rng.choice(["f32", "f32", "bf16", "f16"]),
                     masked=rng.choice([0.0, 0.0, 0.05, 0.3]))
    tokens = spread(rng, 1, 4096)
    io = rng.choice(["same", "same", "f32"])
    # what a chunk costs is its bytes: the widths of a long fp32 chunk stay below the widest
    widest = 4096 if io == "same" or tokens <= 2048 else 2048
    width = lambda: rng.choice([192, 1536, 2048, 4096, spread(rng, 64, 4096)])  # noqa: E731
    d_in, d_out = min(width(), widest), min(width(), widest)
    rank = rng.choice([4, 8, 16, 16, 32, 64, spread(rng, 1, 64)])
    # a batch of decoded tokens has adapters in any order, longer ones come in requests
    mixed = tokens <= 256 and rng.random() < 0.6
    return adapters(None, tokens, d_in, d_out, rank, spread(rng, 1, 2048 // max(rank, 32)),
                    weights=rng.choice(["bf16", "f16"]), io=io, mixed=mixed,
                    run=1 if mixed else spread(rng, 16, 1000), pad=rng.choice([0, 0, 0, 8, 3]))


# ---- inputs ------------------------------------------------------------------

def generator(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def route_inputs(c, seed):
    g = generator(2 * seed, "cuda")
    T, E, t = c["tokens"], c["experts"], DTYPES[c["dtype"]]
    # a router of N(0, 0.02) weights over 4096 normalised values
    logits = (1.28 * torch.randn(T, E, generator=g, device="cuda")).to(t)
    if c["masked"]:
        # pruned experts, the same for every token, and rows of padding with none left
        off = torch.rand(E, generator=g, device="cuda") < c["masked"]
        pad = torch.rand(T, generator=g, device="cuda") < 0.01
        logits[off[None, :] | pad[:, None]] = float("-inf")
    bias = None
    if c["bias"]:
        span = 0.1 if c["score"] == "sigmoid" else 0.01
        bias = span * (2.0 * torch.rand(E, generator=g, device="cuda") - 1.0)
    return logits, bias


def adapter_ids(c, seed):
    """The adapter of each token; every eighth request (about) has none (-1)."""
    g = generator(2 * seed + 1, "cpu")
    T, n = c["tokens"], c["count"]
    order = torch.randperm(n, generator=g).tolist()
    ids, i = [], 0
    while len(ids) < T:
        mean = c["run"]
        length = 1 if c["mixed"] else 1 + int(2 * mean * torch.rand(1, generator=g).item())
        none = i > 0 and torch.rand(1, generator=g).item() < 0.125
        ids += [-1 if none else order[i % n]] * length
        i += 1
    ids = torch.tensor(ids[:T], dtype=torch.int32)
    if c["mixed"]:
        ids = ids[torch.randperm(T, generator=g)]
    return ids


def adapter_inputs(c, seed):
    g = generator(2 * seed + 1, "cuda")
    T, din, dout, r, n = c["tokens"], c["d_in"], c["d_out"], c["rank"], c["count"]
    wt = DTYPES[c["weights"]]
    io = torch.float32 if c["io"] == "f32" else wt
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = rand(T, din + c["pad"]).to(io)[:, :din]
    base = rand(T, dout).to(io)
    a = (rand(n, r, din) / math.sqrt(din)).to(wt)
    b = (0.05 * rand(n, dout, r)).to(wt)
    # alpha / rank, as adapters are trained with
    scale = (2.0 ** torch.randint(-1, 3, (n,), generator=g, device="cuda")).float()
    return x, base, a, b, scale, adapter_ids(c, seed).cuda()


def prepare(case, seed):
    s = {"case": case}
    if case["op"] == "route":
        logits, bias = route_inputs(case, seed)
        s.update(logits=logits, bias=bias)
        if own:
            import hy3_amd as H
            T, k = case["tokens"], case["k"]
            s.update(
                route=H.route_experts,
                spec=H.RouteSpec(n_expert=case["experts"], k=k, score=case["score"],
                                 n_group=case["groups"], topk_group=case["kept"],
                                 group_score=case["best"], renorm=case["renorm"],
                                 scale=case["scale"]),
                ids=torch.empty(T, k, dtype=torch.int32, device="cuda"),
                w=torch.empty(T, k, dtype=torch.float32, device="cuda"))
        return s
    x, base, a, b, scale, ids = adapter_inputs(case, seed)
    s.update(x=x, base=base, ids=ids)
    if not own:
        s.update(a=a, b=b, scale=scale)
        return s
    import hy3_amd as H
    held = H.Adapters(case["count"], case["rank"], case["d_in"], case["d_out"],
                      dtype=case["weights"])
    for i, alpha in enumerate(scale.tolist()):
        held.set(i, a[i], b[i], scale=alpha, on_device=True)
    s.update(held=held, y=torch.empty_like(base),
             io="f32" if case["io"] == "f32" else case["weights"])
    return s


# ---- one pass ----------------------------------------------------------------

def plain_route(case, logits, bias):
    T, E, G = case["tokens"], case["experts"], case["groups"]
    t = DTYPES[case["dtype"]]
    lowest, highest = torch.finfo(t).min, torch.finfo(t).max
    off = ~(logits > lowest)
    if bias is not None:
        off = off | ~(bias > float("-inf"))
    ld = logits.double().clamp(max=highest)
    if case["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-ld))
    else:
        top = torch.where(off, -math.inf, ld).amax(1, keepdim=True)
        e = torch.where(off, 0.0, torch.exp(ld - top))
        s = e / e.sum(1, keepdim=True)
    s = torch.where(off, 0.0, s)
    # without a bias the scores order as the logits do
    key = ld if bias is None else s + bias.double()
    low = torch.finfo(torch.float64).min
    key = torch.where(off, low, key)
    if G > 1:
        members = key.view(T, G, E // G)
        if case["best"] == "max":
            group = members.amax(2)
        else:
            scored = s if bias is None else s + bias.double()
            best = torch.where(off, low, scored).view(T, G, E // G).topk(min(2, E // G), dim=2).values
            second = best[:, :, 1] if best.shape[2] > 1 else torch.full_like(best[:, :, 0], low)
            group = best[:, :, 0] + torch.where(second > low, second, 0.0)
        order = torch.sort(group, dim=1, descending=True, stable=True).indices
        stays = torch.zeros(T, G, dtype=torch.bool, device=key.device)
        stays.scatter_(1, order[:, :case["kept"]], True)
        key = torch.where(stays[:, :, None], members, -math.inf).view(T, E)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :case["k"]]
    w = s.gather(1, ids)
    if case["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return ids.int(), (w * case["scale"]).float()


def plain_adapters(case, x, base, a, b, scale, ids):
    n, r = case["count"], case["rank"]
    u = x.float() @ a.float().view(n * r, -1).t()
    mine = ids[:, None] == torch.arange(n, device=ids.device)
    u = torch.where(mine[:, :, None], u.view(-1, n, r) * scale[None, :, None], 0.0)
    y = base.float() + u.view(-1, n * r) @ b.float().permute(0, 2, 1).reshape(n * r, -1)
    return y.to(base.dtype)


def run(state):
    c = state["case"]
    if c["op"] == "route":
        if not own:
            return plain_route(c, state["logits"], state["bias"])
        state["route"](state["spec"], state["logits"], c["tokens"], state["ids"], state["w"],
                       dtype=c["dtype"], bias=state["bias"],
                       stream=torch.cuda.current_stream().cuda_stream)
        return state["ids"], state["w"]
    if not own:
        return plain_adapters(c, *(state[k] for k in ("x", "base", "a", "b", "scale", "ids")))
    state["held"].apply(state["ids"], state["x"], state["y"], c["tokens"], base=state["base"],
                        x_dtype=state["io"], y_dtype=state["io"],
                        x_stride=c["d_in"] + c["pad"],
                        stream=torch.cuda.current_stream().cuda_stream)
    return state["y"]


def work(case):
    T = case["tokens"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "route":
        E, k = case["experts"], case["k"]
        moved = T * E * size[case["dtype"]] + 8 * T * k + (4 * E if case["bias"] else 0)
        # an exponential, a sum and a comparison per expert, a comparison per choice
        return {"bytes": moved, "flops": T * (12 * E + k * E)}
    io = size["f32" if case["io"] == "f32" else case["weights"]]
    din, dout, r = case["d_in"], case["d_out"], case["rank"]
    used = min(case["count"], T if case["mixed"] else max(1, T // case["run"]))
    moved = io * T * (din + 2 * dout) + 2 * used * r * (din + dout) + 4 * T
    return {"bytes": moved, "flops": 2 * T * r * (din + dout) + T * dout}


# ---- the definition in 64 bits -------------------------------------------------

def exact_route(case, logits, bias):
    """Row by row in numpy: lists sorted by (key descending, index)."""
    import numpy as np
    t = DTYPES[case["dtype"]]
    lowest, highest = torch.finfo(t).min, torch.finfo(t).max
    lg = logits.double().cpu().numpy()
    T, E = lg.shape
    G, k = case["groups"], case["k"]
    size = E // G
    b = None if bias is None else bias.double().cpu().numpy()
    ids = np.empty((T, k), np.int32)
    w = np.empty((T, k), np.float64)
    index = np.arange(E)
    for r in range(T):
        row = np.minimum(lg[r], highest)
        on = row > lowest
        if b is not None:
            on &= b > -np.inf
        s = np.zeros(E)
        if case["score"] == "sigmoid":
            s[on] = 1.0 / (1.0 + np.exp(-row[on]))
        elif on.any():
            e = np.exp(row[on] - row[on].max())
            s[on] = e / e.sum()
        scored = s if b is None else s + b
        key = row if b is None else scored
        allowed = np.ones(E, bool)
        if G > 1:
            rank = []
            for g in range(G):
                here = slice(g * size, (g + 1) * size)
                live = np.sort((key if case["best"] == "max" else scored)[here][on[here]])[::-1]
                if live.size == 0:
                    rank.append((1, 0.0, g))
                else:
                    rank.append((0, -(live[0] if case["best"] == "max" else live[:2].sum()), g))
            allowed[:] = False
            for _, _, g in sorted(rank)[:case["kept"]]:
                allowed[g * size:(g + 1) * size] = True
        rank = np.where(allowed, np.where(on, 0, 1), 2)
        order = np.lexsort((index, -np.where(on, key, 0.0), rank))[:k]
        ids[r] = order
        v = s[order]
        if case["renorm"]:
            v = v / (v.sum() + 1e-20)
        w[r] = v * case["scale"]
    return torch.from_numpy(ids), torch.from_numpy(w)


def exact_adapters(case, x, base, a, b, scale, ids):
    y = base.double().clone()
    for i in range(case["count"]):
        rows = (ids == i).nonzero()[:, 0]
        if rows.numel():
            u = x[rows].double() @ a[i].double().t().contiguous()
            y[rows] += scale[i].double() * (u @ b[i].double().t().contiguous())
    return y


def exact(case, seed):
    if case["op"] == "route":
        return exact_route(case, *route_inputs(case, seed))
    return exact_adapters(case, *adapter_inputs(case, seed))
