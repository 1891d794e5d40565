"""The inputs and bounds of the paged attention's sharper tests, without a GPU: a mistake planted in
the oracle falls outside the bound, and the sizes reach the schedules they are chosen for."""
import pytest
import torch

import paged_bounds as PB
from paged_cases import MANY_UNITS, RISING, SPLIT, TELLING


@pytest.mark.parametrize("kw", SPLIT, ids=str)
def test_a_query_rounded_once_is_outside(kw):
    case = PB.split_case(**kw)
    ref, bound = PB.attention(**case)
    bad, _ = PB.attention(**case, plant="lo")
    T = kw["T"]
    assert ((bad - ref).abs() > 2 * bound)[:, :, :T // 2].any(-1).all()


@pytest.mark.parametrize("kw", TELLING, ids=str)
def test_every_telling_slot_counts(kw):
    case, slots = PB.telling_case(**kw)
    ref, bound = PB.attention(**case)
    T = kw["T"]
    for b, at in enumerate(slots):
        assert len(at) >= min(kw["D"], kw["lens"][b] + T) // 2
        for i, s in enumerate(at):
            if s < case["lens"][b] + T and (ref[b, :, :, i] != 0).any():
                assert (ref[b, :, :, i] > 20 * bound[b, :, :, i])[ref[b, :, :, i] != 0].all()
        context = [i for i, s in enumerate(at) if s < case["lens"][b] and kw.get("window", -1) < 0]
        assert (ref[b][..., context] != 0).all()
    b, i = len(slots) - 1, 0
    bad, _ = PB.attention(**case, hide=(b, slots[b][i]))
    assert ((bad - ref).abs() > bound)[b].any()


@pytest.mark.parametrize("kw", RISING, ids=str)
def test_rows_rescale_and_every_tile_counts(kw):
    """By the kernels' rule (a reference moves when a tile's maximum is more than 2^8 above it) rows move
    finite references, and leaving out the first tile falls outside the bound."""
    case = PB.rising_case(**kw)
    ref, bound = PB.attention(**case)
    H, Hkv, T = kw["H"], kw["Hkv"], kw["T"]
    b = max(range(len(kw["lens"])), key=lambda i: kw["lens"][i])
    L = kw["lens"][b]
    k = PB.O.slot_rows(case["k_cache"], case["table"][b], L + 1, case["k_cache"].shape[0]).repeat_interleave(H // Hkv, 0)
    s = case["q"][b].double() @ k.transpose(1, 2) / 0.6931471805599453
    moved = torch.zeros(H, T)
    now = torch.full((H, T), float("-inf"), dtype=torch.float64)
    for t0 in range(0, L + 1, 64):
        top = s[..., t0:t0 + 64].amax(-1)
        grow = top > now + 8
        moved += grow & now.isfinite()
        now = torch.where(grow, top, now)
    rising = case["q"][b, :, :, 0] != 0
    want = 1 if kw["pattern"] == "end" or kw["step"] <= 8 else 2
    assert rising.any() and (moved[rising] >= min(want, L // 64)).all()
    if kw.get("rows", "all") != "all":
        assert (~rising).any() and (moved[~rising] == 0).all()
    bad, _ = PB.attention(**case, hide=(b, slice(0, 64)))
    assert ((bad - ref).abs() > 2 * bound)[b][rising].any(-1).all()


@pytest.mark.parametrize("kw", MANY_UNITS, ids=lambda kw: f"{kw['dtype']}-{kw['D']}-{kw['T']}-{kw['kind']}".replace("torch.", ""))
def test_ctas_take_several_units(kw):
    """On 148 SMs: CTAs with tiles of two, three and more units, whole ones and parts among them."""
    a = {k: v for k, v in kw.items() if k in ("H", "Hkv", "T", "D", "P", "lens", "kind", "window")}
    segs = PB.segments(B=len(kw["lens"]), **a)
    several = [s for s in segs if len(s) >= 2]
    assert len(several) > 40 and max(map(len, segs)) >= 3
    assert any(k < n for s in several for _, k, n in s) or all(n == 1 for s in several for _, _, n in s)
    assert any(k == n for s in several for _, k, n in s)
