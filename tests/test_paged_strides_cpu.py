"""Strides of the paged cache's axes that are never stepped along do not matter.  Every call has a
later argument that is refused, so that none reaches a launch on any machine."""
import pytest

from test_paged_cpu import CS, _accept, _append, _attend

LATER = {_append: (dict(key=None), "null tensor pointer"), _attend: (dict(ws=128), "256-byte aligned"),
         _accept: (dict(acc=None), "null tensor pointer")}


@pytest.mark.parametrize("call", list(LATER))
@pytest.mark.parametrize("stride", [1 << 31, 1 << 40, 0, -8, 3])
def test_page_stride_of_a_single_page(call, stride):
    """One sequence of 2^21 slots as a contiguous [1, 8, 2^21, 128] cache has a page stride of 2^31."""
    kw, needle = LATER[call]
    s = (stride, CS[1], CS[2])
    rc, msg = call(pages=1, kcs=s, vcs=s, **kw)
    assert rc == -3 and needle in msg, msg


@pytest.mark.parametrize("call", list(LATER))
@pytest.mark.parametrize("name", ["kcs", "vcs"])
@pytest.mark.parametrize("strides", [(1 << 31, CS[1], 128), (CS[0], CS[1], 1 << 31)])
def test_strides_that_are_stepped_along_stay_below_2_to_the_31(call, name, strides):
    rc, msg = call(**{name: strides}, **LATER[call][0])
    assert rc == -3 and "stride too large" in msg, msg
