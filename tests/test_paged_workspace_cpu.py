"""The workspace query of the paged attention and the call agree on what is refused.  Every call
here has a misaligned workspace, so that none passes its checks on any machine."""
import random

import pytest

import rdnattention_b200 as R
from test_paged_cpu import _attend

GOOD = dict(B=2, H=8, Hkv=8, T=3, D=128, P=64, mp=4)
SIZE_ERRORS = ("empty problem", "unsupported head_dim", "unsupported page_size", "exceeds 2^30", "too many heads",
               "positive multiple", "sequence too long", "too large for one launch")


def _size(a):
    return R._lib_handle().rdna_attention_paged_workspace_size(a["B"], a["H"], a["Hkv"], a["T"], a["D"], a["P"], a["mp"])


def _call(a, wsb):
    s = (1 << 30, 256, 256)  # strides: valid for every size, so that no other check speaks first
    return _attend(**a, qs=(1 << 38, 256, 256), os=(1 << 38, 256, 256), kcs=s, vcs=s, pages=8, ts=a["mp"], ws=128,
                   wsb=wsb)


@pytest.mark.parametrize("kw", [
    dict(B=0), dict(B=(1 << 24) + 1), dict(Hkv=0), dict(Hkv=65536, H=65536), dict(H=0), dict(H=12), dict(D=0), dict(D=40),
    dict(D=288), dict(P=0), dict(P=4), dict(P=12), dict(P=48), dict(mp=0), dict(mp=1 << 25), dict(P=1 << 31, mp=1),
    dict(T=1 << 29), dict(T=262144, H=16), dict(T=65537, D=256), dict(T=262144, Hkv=65535, H=65535, mp=1 << 24)], ids=str)
def test_sizes_the_call_refuses_have_no_workspace(kw):
    a = {**GOOD, **kw}
    assert _size(a) == 0
    rc, msg = _call(a, 1 << 40)
    assert rc == -3 and any(e in msg for e in SIZE_ERRORS), msg


@pytest.mark.parametrize("kw", [dict(), dict(T=262144), dict(T=65536, D=256), dict(P=8), dict(P=65), dict(mp=1 << 24),
                                dict(B=1 << 24), dict(D=32)], ids=str)
def test_sizes_at_the_limits_have_one(kw):
    a = {**GOOD, **kw}
    n = _size(a)
    assert n > 0
    assert "workspace missing" in _call(a, n - 1)[1]
    assert "256-byte aligned" in _call(a, n)[1]


def test_query_and_call_agree_on_drawn_sizes():
    rng = random.Random(5)
    for _ in range(3000):
        Hkv = rng.choice([0, 1, 2, 8, 65535, 65536])
        a = dict(B=rng.choice([0, 1, 7, 4000, 1 << 24, 1 << 25]), Hkv=Hkv, H=Hkv * rng.choice([0, 1, 5, 64]) + rng.choice([0, 0, 0, 1]),
                 T=rng.choice([1, 17, 2000, 65536, 1 << 18, 1 << 28]), D=rng.choice([32, 40, 128, 160, 256, 512]),
                 P=rng.choice([4, 8, 24, 64, 100, 1 << 20, 1 << 30]), mp=rng.choice([0, 1, 300, 1 << 22, 1 << 27]))
        n = _size(a)
        msg = _call(a, max(n, 1))[1]
        assert (n == 0) == any(e in msg for e in SIZE_ERRORS) and (n == 0 or "256-byte aligned" in msg), (a, n, msg)
