"""hy3x_linear4_apply: how far fp32 outputs are from the definition in 64 bits, where the
tolerances of test_linear4.py (in steps of the sum of all magnitudes) say little: x of one
sign, whose sums with the integers of the weights nearly cancel.

The root mean square of the errors may be that of the roundings which a sum of centred
operands cannot do without, each independent of the others and by whichever rule it goes, up
to a whole step of 2^-23 of what it rounds, so of a root mean square of 2^-23 / sqrt(3) of it:
 - for each run of 32 inputs and part of x (fp32: three), the sum of the group's products
   (q - 7.5) x so far, or its largest product;
 - likewise the sum of the group's x so far, times z - 7.5 (8 - 7.5 without zero points);
 - for each group, two additions to the row's running sum, with the one or the other there;
 - four joins of waves at the sum's size, and the output's rounding."""
import pytest

import hy3_amd as H
from test_linear4 import held, pack, torch  # noqa: F401 (a fixture)

STEP = 2.0 ** -23 / 3 ** 0.5


def weights(torch, d_out, d_in, group, zeros, seed):
    """q of N(z, 2.5), as a quantiser leaves them: rows of W have no sign of their own."""
    g = torch.Generator().manual_seed(seed)
    groups = -(-d_in // group)
    s = (0.008 * torch.exp(0.3 * torch.randn(d_out, groups, generator=g))).bfloat16()
    z = torch.full((d_out, groups), 8.0)
    if zeros:
        z = (z + torch.randn(d_out, groups, generator=g)).round().clamp(0, 15)
    of = torch.arange(d_in) // group
    q = (z[:, of] + 2.5 * torch.randn(d_out, d_in, generator=g)).round().clamp(0, 15)
    return q.to(torch.uint8), s, z.to(torch.uint8) if zeros else None


def activations(torch, kind, T, d_in, seed):
    x = torch.randn(T, d_in, generator=torch.Generator().manual_seed(seed))
    return {"both signs": x, "one sign": x.abs(), "far from 0": x + 10.0}[kind]


def allowed(torch, q, s, z, group, x, parts):
    """The exact outputs, and the root mean square of their errors."""
    T, d_in = x.shape
    d_out, groups = s.shape
    qd = q.double() - 7.5
    zd = (torch.full(s.shape, 8.0, dtype=torch.float64) if z is None else z.double()) - 7.5
    sd = s.double()
    y = torch.zeros(T, d_out, dtype=torch.float64)
    var = torch.zeros(T, d_out, dtype=torch.float64)
    for g in range(groups):
        dot = torch.zeros(T, d_out, dtype=torch.float64)
        total = torch.zeros(T, 1, dtype=torch.float64)
        of_dot, of_total = torch.zeros_like(dot), torch.zeros_like(total)
        for k in range(g * group, min((g + 1) * group, d_in), 32):
            n = slice(k, min(k + 32, (g + 1) * group, d_in))
            a, b = qd[:, n], x[:, n]
            most = b.abs().amax(1, keepdim=True)
            before, dot = dot, dot + b @ a.t()
            size = torch.maximum(torch.maximum(before.abs(), dot.abs()),
                                 most * a.abs().amax(1)[None])
            of_dot += parts * size ** 2
            before, total = total, total + b.sum(1, keepdim=True)
            of_total += parts * torch.maximum(torch.maximum(before.abs(), total.abs()), most) ** 2
        scale, off = sd[:, g][None], (sd * zd)[:, g][None]
        was, y = y, y + scale * dot - off * total
        size = torch.stack((was, y, was + scale * dot, was - off * total)).abs().amax(0)
        var += (scale ** 2 * of_dot + off ** 2 * of_total + 2 * size ** 2) * STEP ** 2
    var += 5 * (y * STEP) ** 2
    return y, var.mean().sqrt().item()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["both signs", "one sign", "far from 0"])
@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,d_in,d_out,group", [
    (1, 4096, 512, 128), (4, 4096, 13000, 64), (12, 2048, 512, 64), (20, 1024, 512, 32),
    (64, 4096, 700, 128), (130, 1536, 2048, 32), (300, 2000, 512, 64)])
def test_errors_of_outputs(torch, T, d_in, d_out, group, x, kind):  # noqa: F811
    types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    rows = slice(d_out - 500, d_out)  # the ones that are looked at
    for zeros in (False, True):
        q, s, z = weights(torch, d_out, d_in, group, zeros, d_in + T)
        h = held(d_out, d_in, group, "bf16", q, s, z, pack(q, torch))
        xs = activations(torch, kind, T, d_in, T).to(types[x])
        y = torch.empty(T, d_out, device="cuda")
        h.apply(xs.cuda(), y, T)
        n = slice(max(T - 16, 0), T)
        exact, most = allowed(torch, q[rows], s[rows], z if z is None else z[rows], group,
                              xs[n].double(), 3 if x == "f32" else 1)
        off = (y[n, rows].double().cpu() - exact).square().mean().sqrt().item()
        assert off <= most, (zeros, off / most)
        h.close()
