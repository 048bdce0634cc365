"""hy3x_logprobs: relative errors where one token has nearly all of a row's mass, and the root
mean square of the errors over long rows.

With d = l - max l and R the sum of e^d over the other tokens, log p of the best one is
-log(1 + R) and the entropy log(1 + R) + sum |d| e^d / (1 + R): sums of terms of one sign.
Each e^d is relatively off by (2 |d| + 4) roundings of 2^-24 (as in test_logprobs.py), |d| by one
more; a sum passes at most V / 256 + 8 additions in fp32; the result is rounded once."""
import numpy as np
import pytest

import hy3_amd as H
from test_logprobs import HALF, NAMES, Call, given, logits, torch  # noqa: F401 (a fixture)


def exact(l, lowest):
    """-log p of the best token, entropy, R and the largest |d|, in 64 bits; one best token."""
    l = l.astype(np.float64)
    m = l.max(1, keepdims=True)
    d = np.where(l > lowest, l - m, -np.inf)
    d[np.arange(len(l)), l.argmax(1)] = -np.inf
    e = np.exp(d)
    R = e.sum(1)
    away = np.where(np.isneginf(d), 0.0, -d)
    return np.log1p(R), np.log1p(R) + (away * e).sum(1) / (1 + R), R, away.max(1)


def check_peaks(torch, l, top):  # noqa: F811
    T, V = l.shape
    call = Call(torch, l, l.float().argmax(1).int(), top)()
    best, entropy, R, far = exact(l.float().cpu().numpy(), torch.finfo(l.dtype).min)
    assert (R < 0.06).all()
    tol = (V / 256 + 8 + 2 * far + 8) * HALF
    for what, got, want in (("logp", -call.logp, best), ("entropy", call.entropy, entropy),
                            ("top_logp", -call.best[:, 0], best)):
        got = got.double().cpu().numpy()
        off = np.abs(got - want) / want
        assert (off <= tol).all(), (what, off.max(), tol[off.argmax()], got[:5], want[:5])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
@pytest.mark.parametrize("V", [2, 3, 5, 16, 40, 700])
def test_peaks_of_short_rows(torch, V, kind):  # noqa: F811
    """The others are few, and lie with the best one in one lane's logits or beside them."""
    T = 62
    l = torch.zeros(T, V)
    l[torch.arange(T), torch.arange(T) % V] = torch.linspace(10.0, 40.5, T)
    l += logits(torch, T, V, "f32", V, spread=0.25).cpu()
    check_peaks(torch, l.to(getattr(torch, NAMES[kind])).cuda(), 1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
@pytest.mark.parametrize("T,V", [(1, 120832), (30, 120832), (300, 5000), (200, 32003), (600, 9000)])
def test_peaks_of_long_rows(torch, T, V, kind):  # noqa: F811
    """All others have a part, or a few, or only some beside the best one."""
    t = getattr(torch, NAMES[kind])
    l = logits(torch, T, V, "f32", V, spread=0.25).clone()
    at = given(torch, T, V, 5).long()
    rows = torch.arange(T, device="cuda")
    l[rows, at] = torch.linspace(16.0, 42.0, T, device="cuda")
    check_peaks(torch, l.to(t), 3)
    few = torch.full_like(l, float("-inf"))
    for step in (1, 8, 255, 256, 2048):
        near = (at + step) % V
        few[rows, near] = l[rows, near]
    few[rows, at] = l[rows, at]
    check_peaks(torch, few.to(t), 2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(NAMES))
@pytest.mark.parametrize("T", [60, 300, 600])
def test_errors_of_long_rows(torch, T, kind):  # noqa: F811
    """A lane's sum takes its logits a batch of 16 at a time, 30 batches or so: of a relative
    2^-24 for each addition at most 2^-24 / sqrt(3) remains in the mean of squares, divided over
    256 lanes or more; so that the rounding of the outputs themselves (at most half a step of
    them, 2^-24 / sqrt(3) in the mean of squares) is nearly all of their errors."""
    V = 120832
    l = logits(torch, T, V, kind, T)
    tokens = given(torch, T, V, T)
    call = Call(torch, l, tokens, 0)()
    lp = torch.log_softmax(l.double(), 1)
    entropy = -(lp.exp() * lp).sum(1)
    logp = lp.gather(1, tokens.long()[:, None])[:, 0]
    for what, got, want in (("logp", call.logp, logp), ("entropy", call.entropy, entropy)):
        off = ((got.double() - want) / want).square().mean().sqrt().item()
        assert off <= HALF, (what, off / HALF)
