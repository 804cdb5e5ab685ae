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


def test_outputs_apart_from_inputs():
    """The last refusal: in place, or overlapping by an element, in both forms."""
    need = J.lib().jero_hip_verify_drafts_workspace_bytes(2, 100000)
    a = dict(target=FAKE, draft=FAKE, tokens=0x20000, starts=0x21000, granted=0x22000, u=0x23000, ul=0x24000, out=0x25000,
             acc=0x26000, dropped=0x27000, size=need)
    lengths = dict(tokens=6, starts=3, granted=2, u=4, ul=2)
    for V in (100, 100000):
        for o, n in (("out", 6), ("acc", 2), ("dropped", 2)):
            for i, m in lengths.items():
                for at in (a[i], a[i] + 4 * (m - 1), a[i] - 4 * (n - 1)):
                    assert verify(**dict(a, V=V, **{o: at})) == 21, (o, i, at)
                    assert "overlaps" in J.lib().jero_hip_last_error().decode()
