"""Products of 4-bit weights and log-probabilities of tokens, as measurable cases.

Two operators of a served model around its MoE FFN blocks:

  linear4    hy3_amd.Linear4: y = base + W x for a matrix of 4-bit weights with
             a scale, and perhaps a zero point, for each group of a row's weights:
             the projections beside which adapters stand, and the LM head;
  logprobs   hy3_amd.logprobs: of the head's logits, the log-probability of each
             row's given token, the row's entropy and its most probable tokens.

Where `own` is false, run() computes them in their plain form: elementary torch
operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
VOCAB = 120832  # rows of the LM head


def linear4(name, tokens, d_in, d_out, group=128, scales="bf16", zeros=False, x="bf16", y="bf16",
            base=False, pad=0):
    """zeros: a zero point for each group (else 8). base: added to the product. pad:
    elements between the rows of x."""
    c = {"op": "linear4", "tokens": tokens, "d_in": d_in, "d_out": d_out, "group": group,
         "scales": scales, "zeros": zeros, "x": x, "y": y, "base": base, "pad": pad}
    return dict(c, name=name) if name else c


def logprobs(name, tokens, vocab, top=0, dtype="f32", entropy=True, masked=0.0, pad=0):
    """masked: the share of the vocabulary that a grammar rules out. pad: elements
    between the rows."""
    c = {"op": "logprobs", "tokens": tokens, "vocab": vocab, "top": top, "dtype": dtype,
         "entropy": entropy, "masked": masked, "pad": pad}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoded token: attention's output projection, added to the residual stream
        linear4("linear4_1_out", 1, 8192, 4096, base=True),
        # the LM head for one decoded token, fp32 activations and logits
        linear4("linear4_1_head", 1, 4096, VOCAB, x="f32", y="f32"),
        # odd everything: tokens, widths, the last group, rows of a wider buffer
        linear4("linear4_7_odd", 7, 1001, 777, group=32, scales="f16", zeros=True, x="f16",
                y="f16", pad=3),
        # a decode batch's projection, weights with zero points
        linear4("linear4_16_in", 16, 4096, 8192, group=64, scales="f16", zeros=True, x="f16",
                y="f16"),
        # the LM head for a decode batch
        linear4("linear4_64_head", 64, 4096, VOCAB, y="f32"),
        # a ragged prefill chunk on fp32 activations, small groups
        linear4("linear4_300_f32", 300, 1536, 4096, group=32, scales="f16", zeros=True, x="f32",
                y="f32", base=True),
        # the longest prefill chunk
        linear4("linear4_2048", 2048, 4096, 8192),
        # the token that one sequence decoded, with alternatives for its answer
        logprobs("logprobs_1", 1, VOCAB, top=20),
        # a decode batch
        logprobs("logprobs_64", 64, VOCAB, top=5),
        # constrained decoding over an odd vocabulary, rows of a wider buffer
        logprobs("logprobs_333_masked", 333, 32003, top=8, dtype="bf16", masked=0.9, pad=5),
        # scored text with alternatives
        logprobs("logprobs_511", 511, 50021, top=20, dtype="f16"),
        # the largest: a long prompt scored
        logprobs("logprobs_2048", 2048, VOCAB, dtype="bf16"),
    ]


def spread(rng, low, high):
    """A whole number in [low, high], even over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    if rng.random() < 0.55:
        width = lambda most: rng.choice([1536, 4096, 8192, spread(rng, 64, most)])  # noqa: E731
        d_in = width(8192)
        d_out = VOCAB if rng.random() < 0.15 else width(16384)
        x = rng.choice(["bf16", "bf16", "f16", "f32"])
        # fp32 activations cost their products three times over
        most = 2048 * 4096 * 8192 // (3 if x == "f32" else 1)
        if d_in * d_out > VOCAB * 4096:
            d_in = 4096
        tokens = min(spread(rng, 1, 4096), max(1, most // (d_in * d_out)))
        return linear4(None, tokens, d_in, d_out, group=rng.choice([32, 64, 128, 128]),
                       scales=rng.choice(["f16", "bf16"]), zeros=rng.random() < 0.5, x=x,
                       y=rng.choice([x, x, "f32"]), base=rng.random() < 0.4,
                       pad=rng.choice([0, 0, 0, 8, 3]))
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    vocab = rng.choice([VOCAB, 32003, spread(rng, 1000, 150000)])
    tokens = min(spread(rng, 1, 4096), 2048 * VOCAB // (vocab * (2 if dtype == "f32" else 1)))
    top = rng.choice([0, 1, 5, 8, 20, rng.randint(1, 32)])
    if top:  # ordering alternatives costs the plain form most
        tokens = min(tokens, 1024)
    return logprobs(None, tokens, vocab, top=top, dtype=dtype, entropy=rng.random() < 0.8,
                    masked=rng.choice([0.0, 0.0, 0.5, 0.9]), pad=rng.choice([0, 0, 8, 5]))


# ---- inputs ------------------------------------------------------------------

def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def linear4_inputs(c, seed):
    g = generator(2 * seed)
    T, din, dout = c["tokens"], c["d_in"], c["d_out"]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    groups = -(-din // c["group"])
    # weights of N(0, 0.02), rounded to steps of about a sixth of their group's span
    scales = (0.02 / 2.5 * torch.exp(0.3 * rand(dout, groups))).to(DTYPES[c["scales"]])
    zeros = None
    if c["zeros"]:
        zeros = (8 + rand(dout, groups)).round().clamp(0, 15).to(torch.uint8)
    half = -(-din // 2)
    packed = torch.empty(dout, half, dtype=torch.uint8, device="cuda")
    for rows in packed.split(16384):
        q = (8 + 2.5 * rand(rows.shape[0], 2 * half)).round().clamp(0, 15).to(torch.uint8)
        rows.copy_(q[:, 0::2] | q[:, 1::2] << 4)
    # normalised activations, a few channels of which stand out
    x = rand(T, din + c["pad"]) * torch.where(rand(din + c["pad"]) > 2.5, 8.0, 1.0)
    x = x.to(DTYPES[c["x"]])[:, :din]
    base = rand(T, dout).to(DTYPES[c["y"]]) if c["base"] else None
    return packed, scales, zeros, x, base


def logprobs_inputs(c, seed):
    g = generator(2 * seed + 1)
    T, V, t = c["tokens"], c["vocab"], DTYPES[c["dtype"]]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    logits = 2.0 * rand(T, V + c["pad"])
    # a few candidates stand out, in some rows one of them alone
    likely = torch.randint(0, V, (T, 1), generator=g, device="cuda")
    likely = (likely + torch.arange(12, device="cuda") * (V // 12)) % V
    logits.scatter_(1, likely, 9.0 + 3.0 * rand(T, 12))
    tokens = torch.where(rand(T) < 1.0, likely[:, 0],
                         torch.randint(0, V, (T,), generator=g, device="cuda"))
    logits = logits.to(t)
    if c["masked"]:
        off = torch.rand(V + c["pad"], generator=g, device="cuda") < c["masked"]
        off = off.repeat(T, 1).scatter_(1, tokens[:, None], False)
        logits[off] = float("-inf")
    # rows of padding have no token
    tokens = torch.where(rand(T) > 2.3, -1, tokens) if T > 1 else tokens
    return logits[:, :V], tokens.int()


def prepare(case, seed):
    s = {"case": case}
    if case["op"] == "linear4":
        packed, scales, zeros, x, base = linear4_inputs(case, seed)
        s.update(x=x, base=base)
        if not own:
            s.update(packed=packed, scales=scales, zeros=zeros)
            return s
        import hy3_amd as H
        held = H.Linear4(case["d_out"], case["d_in"], group=case["group"], dtype=case["scales"])
        held.set(packed, scales, zeros, on_device=True)
        y = torch.empty(case["tokens"], case["d_out"], dtype=DTYPES[case["y"]], device="cuda")
        s.update(held=held, y=y)
        return s
    logits, tokens = logprobs_inputs(case, seed)
    s.update(logits=logits, tokens=tokens)
    if own:
        import hy3_amd as H
        T, top = case["tokens"], case["top"]
        f32 = lambda *n: torch.empty(*n, dtype=torch.float32, device="cuda")  # noqa: E731
        s.update(call=H.logprobs, logp=f32(T), entropy=f32(T) if case["entropy"] else None,
                 top_ids=torch.empty(T, top, dtype=torch.int32, device="cuda") if top else None,
                 top_logp=f32(T, top) if top else None)
        room = H.logprobs_workspace(T, case["vocab"], top)
        s["workspace"] = torch.empty(room, dtype=torch.uint8, device="cuda") if room else None
    return s


# ---- one pass ----------------------------------------------------------------

def plain_linear4(c, packed, scales, zeros, x, base):
    q = torch.stack((packed & 15, packed >> 4), 2).view(c["d_out"], -1)[:, :c["d_in"]].float()
    of = torch.arange(c["d_in"], device="cuda") // c["group"]
    w = q - (8.0 if zeros is None else zeros.float()[:, of])
    y = x.float() @ (w * scales.float()[:, of]).t()
    if base is not None:
        y = y + base.float()
    return y.to(DTYPES[c["y"]])


def plain_logprobs(c, logits, tokens):
    t = DTYPES[c["dtype"]]
    l = logits.float().clamp(max=torch.finfo(t).max) + 0.0
    off = ~(l > torch.finfo(t).min)
    m = torch.where(off, torch.finfo(torch.float32).min, l).amax(1, keepdim=True)
    away = torch.where(off, 0.0, l - m)
    e = torch.where(off, 0.0, torch.exp(away))
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    mine = tokens.clamp(min=0).long()[:, None]
    given = torch.where(off.gather(1, mine), -math.inf, away.gather(1, mine) - lse)
    out = [torch.where(tokens < 0, 0.0, given[:, 0])]
    if c["entropy"]:
        out.append((lse - (e * away).sum(1, keepdim=True) / total)[:, 0])
    if c["top"]:
        # the values' bits in their order, before the index: no two keys are equal
        bits = torch.where(off, -math.inf, l).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7fffffff)).long() << 32
        key = key - torch.arange(l.shape[1], device="cuda")
        ids = key.topk(c["top"], dim=1).indices
        out += [ids.int(), torch.where(off.gather(1, ids), -math.inf, away.gather(1, ids) - lse)]
    return tuple(out)


def run(state):
    c = state["case"]
    if c["op"] == "linear4":
        if not own:
            return plain_linear4(c, *(state[k] for k in ("packed", "scales", "zeros", "x", "base")))
        state["held"].apply(state["x"], state["y"], c["tokens"], base=state["base"],
                            stream=torch.cuda.current_stream().cuda_stream)
        return state["y"]
    if not own:
        return plain_logprobs(c, state["logits"], state["tokens"])
    state["call"](state["logits"], state["tokens"], c["tokens"], state["logp"],
                  entropy=state["entropy"], top_ids=state["top_ids"], top_logp=state["top_logp"],
                  workspace=state["workspace"], stream=torch.cuda.current_stream().cuda_stream)
    out = [state["logp"]]
    if c["entropy"]:
        out.append(state["entropy"])
    if c["top"]:
        out += [state["top_ids"], state["top_logp"]]
    return tuple(out)


def work(case):
    T = case["tokens"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "linear4":
        din, dout = case["d_in"], case["d_out"]
        groups = -(-din // case["group"])
        moved = dout * (-(-din // 2) + groups * (3 if case["zeros"] else 2))
        moved += T * (din * size[case["x"]] + dout * size[case["y"]] * (2 if case["base"] else 1))
        return {"bytes": moved, "flops": 2 * T * din * dout}
    V, top = case["vocab"], case["top"]
    moved = T * (V * size[case["dtype"]] + 8 + (4 if case["entropy"] else 0) + 8 * top)
    # difference, exponential, sum; product and sum of the entropy; a comparison
    return {"bytes": moved, "flops": T * V * (4 + (2 if case["entropy"] else 0) + (1 if top else 0))}


# ---- the definition in 64 bits -------------------------------------------------

def exact_linear4(c, packed, scales, zeros, x, base):
    """Group by group: scale (x q - zero sum x), for a few thousand rows of W at a time."""
    g, din = c["group"], c["d_in"]
    xd = x.double()
    out = []
    for first in range(0, c["d_out"], 8192):
        rows = slice(first, first + 8192)
        p = packed[rows].long()
        y = torch.zeros(c["tokens"], p.shape[0], dtype=torch.float64, device="cuda")
        for k in range(0, din, g):
            index = torch.arange(k, min(k + g, din), device="cuda")
            q = (p[:, index // 2] >> (4 * (index % 2))) & 15
            part = xd[:, index]
            s = scales[rows, k // g].double()
            z = 8.0 if zeros is None else zeros[rows, k // g].double()
            y += (part @ q.double().t().contiguous() - part.sum(1, keepdim=True) * z) * s
        out.append(y)
    y = torch.cat(out, 1)
    return y if base is None else y + base.double()


def exact_logprobs(c, logits, tokens):
    t = DTYPES[c["dtype"]]
    lowest, highest = torch.finfo(t).min, torch.finfo(t).max
    logp, entropy, ids, best = [], [], [], []
    for l, token in zip(logits.split(64), tokens.split(64)):
        l = l.double().clamp(max=highest) + 0.0
        l = torch.where(l > lowest, l, -math.inf)
        lp = l - torch.logsumexp(l, 1, keepdim=True)
        mine = lp.gather(1, token.clamp(min=0).long()[:, None])[:, 0]
        logp.append(torch.where(token < 0, 0.0, mine))
        entropy.append(-(lp.exp() * torch.where(lp > -math.inf, lp, 0.0)).sum(1))
        if c["top"]:
            order = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :c["top"]]
            ids.append(order.int())
            best.append(lp.gather(1, order))
    out = [torch.cat(logp)]
    if c["entropy"]:
        out.append(torch.cat(entropy))
    if c["top"]:
        out += [torch.cat(ids), torch.cat(best)]
    return tuple(out)


def exact(case, seed):
    if case["op"] == "linear4":
        return exact_linear4(case, *linear4_inputs(case, seed))
    return exact_logprobs(case, *logprobs_inputs(case, seed))
