"""hy3x_logprobs_workspace: a workspace that is sized once, for the largest batch."""
import pytest

import hy3_amd as H
from test_logprobs import Call, check, given, logits, torch  # noqa: F401 (a fixture)


@pytest.mark.parametrize("V", [1, 2048, 30000, 32003, 50021, 64000, 120832, 1000000, 1 << 24])
def test_no_batch_needs_more_than_a_larger_one(V):
    for top in {0, min(V, 5), min(V, 32)}:
        need = [H.logprobs_workspace(T, V, top) for T in range(1, 1100)]
        assert need == sorted(need)
        assert need[-1] == H.logprobs_workspace(1 << 24, V, top)


def test_a_call_accepts_what_a_larger_batch_was_told():
    """Too little is refused before the launch; what a batch of 256 was told is not."""
    lib = H.lib()
    for V in (64000, 120832, 1 << 20, 1 << 24):
        room = H.logprobs_workspace(256, V, 20)
        for T in (*range(1, 140), 159, 160, 200, 255, 256):
            for kind in (0, 1, 2):
                # the outputs overlap: refused for that, after the workspace was looked at
                rc = lib.hy3x_logprobs(1 << 40, kind, V, V, 1 << 20, T, 20, 1 << 20, 1 << 21,
                                       1 << 22, 1 << 23, 1 << 24, room, None)
                assert rc == -1 and b"overlaps" in lib.hy3x_last_error(), (V, T, kind)


@pytest.mark.gpu
def test_one_workspace_for_every_batch(torch):  # noqa: F811
    V, top = 120832, 20
    room = H.logprobs_workspace(256, V, top)
    ws = torch.empty(room, dtype=torch.uint8, device="cuda") if room else None
    l, tokens = logits(torch, 256, V, "bf16", 1), given(torch, 256, V, 1)
    for T in (1, 7, 60, 64, 66, 90, 256):
        call = Call(torch, l[:T], tokens[:T], top)
        call.ws = ws
        check(torch, call())


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,kind", [(100, 120832, "f32"), (140, 120832, "bf16"),
                                      (20, 500000, "f16"), (258, 32003, "bf16")])
def test_rows_in_parts(torch, T, V, kind):  # noqa: F811
    """As many rows as are split, a few more, and longer ones; masked parts among them."""
    l = logits(torch, T, V, kind, 2).clone()
    l[3, V // 3:] = float("-inf")
    l[4, :V // 2] = float("nan")
    l[5] = float("-inf")
    l[6] = float("-inf")
    l[6, V - 2:] = 1.0
    check(torch, Call(torch, l, given(torch, T, V, 3), 20)())
