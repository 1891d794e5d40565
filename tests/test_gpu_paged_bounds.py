"""The paged attention on the GPU within the bound that its hi + lo query allows (paged_bounds.py),
on inputs on which single slots, low bits of the query, rescales of O and the state carried from unit
to unit count."""
import pytest
import torch

import paged_bounds as PB
from paged_cases import MANY_UNITS, RISING, SPLIT, TELLING
from test_gpu_paged import CASES

pytestmark = pytest.mark.gpu

R = pytest.importorskip("rdnattention_b200")


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    assert R.debug_read_status() == (0, 0), "a kernel recorded an expired wait"


def attend(q, k_cache, v_cache, table, lens, news=None, mask=None, positions=None, cos=None, sin=None, window=-1,
           scale=None):
    def cuda(t):
        return None if t is None else t.cuda()

    def ints(x):
        return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")

    return R.flash_attn_paged(cuda(q), cuda(k_cache), cuda(v_cache), cuda(table), ints(lens), new_lens=ints(news),
                              tree_mask=cuda(mask), positions=cuda(positions), rot_cos=cuda(cos), rot_sin=cuda(sin),
                              window_size=window, scale=scale)


def check(case):
    ref, bound = PB.attention(**case)
    got = attend(**case)
    err = (got.double().cpu() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside; worst {(err / bound).max().item():.3g} bounds"
    return got


def _id(kw):
    return "-".join(str(v).replace("torch.", "").replace(" ", "")[:40] for v in kw.values())


@pytest.mark.parametrize("kw", SPLIT, ids=_id)
def test_low_bits_of_the_turned_query(kw):
    check(PB.split_case(**kw))


@pytest.mark.parametrize("kw", TELLING, ids=_id)
def test_single_slots(kw):
    check(PB.telling_case(**kw)[0])


@pytest.mark.parametrize("kw", RISING, ids=_id)
def test_rising_maxima(kw):
    check(PB.rising_case(**kw))


@pytest.mark.parametrize("kw", MANY_UNITS, ids=_id)
def test_several_units_per_cta(kw):
    """Twice: what one unit leaves to the next does not depend on timing."""
    case = PB.plain_case(**kw)
    assert torch.equal(check(case), attend(**case))


@pytest.mark.parametrize("pattern,rows", [("every", "odd"), ("second", "warps"), ("end", "all")])
def test_several_units_with_rising_maxima(pattern, rows):
    """A reference and a sum of the unit before must not reach the next one."""
    lens = [(i * 97) % 460 for i in range(40)]
    case = PB.rising_case(PB.BF16, 16, 8, 40, 64, 64, lens, pattern, 10, rows)
    assert max(len(s) for s in PB.segments(40, 16, 8, 40, 64, 64, lens)) >= 3
    check(case)


@pytest.mark.parametrize("kw", CASES, ids=_id)
def test_random_inputs(kw):
    check(PB.plain_case(**{k: v for k, v in kw.items() if k != "order"}))


@pytest.mark.parametrize("T,kind,window", [(1, "chain", -1), (4, "chain", 70), (16, "tree", 90), (64, "tree", -1)])
@pytest.mark.parametrize("length", [0, 64, 700, 6001])
@pytest.mark.parametrize("dtype,H,Hkv,D,P", [(PB.F16, 32, 8, 128, 64), (PB.BF16, 24, 12, 64, 16), (PB.F16, 8, 8, 256, 72)])
def test_single_sequence(T, kind, window, length, dtype, H, Hkv, D, P):
    check(PB.plain_case(dtype, H, Hkv, T, D, P, [length], kind, window))
