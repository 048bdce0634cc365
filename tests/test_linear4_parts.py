"""hy3x_linear4_apply of fp32 x whose values need all three of its two-byte parts: in the
kernel that holds x in registers (up to 4 tokens of a wide output, groups of 64 and 128) and
in every shape of tiles.

A token has one number: an odd one between 2^19 and 2^20, of which the last part is never 0
and the second hardly ever. Its products with 2 q - 15 are whole numbers below 2^24, those with
2 zero - 15 meet them in one FMA, and the difference is again below 2^24 (at 2^24 an even
number), so that the outputs are exact; a part that is lost, or met by other weights, shows.
"""
import pytest

import hy3_amd as H
from test_linear4 import SHAPES, torch  # noqa: F401 (a fixture)


def exact_outputs(torch, T, d_in, d_out, group, trials):  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(T + d_in)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda")
    packed = whole(0, 256, d_out, (d_in + 1) // 2).to(torch.uint8)
    groups = -(-d_in // group)
    z = whole(0, 17, d_out, groups).to(torch.uint8)
    s = (2.0 ** (whole(0, 3, d_out, groups) - 1)).bfloat16()
    h = H.Linear4(d_out, d_in, group=group, dtype="bf16")
    h.set(packed, s, z, on_device=True)
    for trial in range(trials):
        k = whole(0, d_in, T)
        if trial == 0:
            k[0], k[-1] = 0, d_in - 1
        value = (whole(0, 1 << 18, T) * 2 + 1 + (1 << 19)) * (whole(0, 2, T) * 2 - 1)
        x = torch.zeros(T, d_in, device="cuda")
        x[torch.arange(T, device="cuda"), k] = value.float()
        assert torch.equal(x.sum(1).long(), value)
        y = torch.full((T, d_out), 5.0, device="cuda")
        h.apply(x, y, T)
        q = (packed[:, k // 2] >> (4 * (k % 2))[None].to(torch.uint8)) & 15
        want = (q.long() - z[:, k // group].long()) * value[None] * s[:, k // group].double()
        assert torch.equal(y.double(), want.t()), (trial, k.tolist()[:5])
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("d_in", [2049, 2500, 3333, 4096])
@pytest.mark.parametrize("T", [1, 2, 3, 4])
def test_parts_in_registers(torch, T, d_in, group):  # noqa: F811
    exact_outputs(torch, T, d_in, 12600, group, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,d_in,d_out", SHAPES)
def test_parts_in_every_shape(torch, T, d_in, d_out, group):  # noqa: F811
    exact_outputs(torch, T, d_in, d_out, group, 3 if T > 16 else 12)
