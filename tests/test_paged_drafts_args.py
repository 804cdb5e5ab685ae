"""Refusals of verify_drafts' forms, without a GPU: nothing is enqueued and no pointer is followed."""
import jero_hip as J

FAKE = 0x10000


def verify(target=FAKE, ts=100000, draft=FAKE, ds=100000, tokens=FAKE, starts=FAKE, granted=FAKE, u=FAKE, ul=FAKE, n=2, T=6, N=4,
           V=100000, out=FAKE + 4096, acc=FAKE, dropped=None, ws=FAKE, size=31):
    return J.lib().jero_hip_verify_drafts_granted(target, ts, draft, ds, tokens, starts, granted, u, ul, n, T, N, V, out, acc,
                                                  dropped, ws, size, None)


def test_granted():
    assert verify(granted=FAKE + 2) == 21
    for granted in (None, FAKE):  # (a workspace that is too small is refused last)
        assert verify(granted=granted) == 14
        assert "workspace" in J.lib().jero_hip_last_error().decode()
    assert verify(out=None) == 21 and verify(n=0) == 14
