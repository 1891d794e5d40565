"""Values that are not finite, or hardly: NaN and infinities in the query and in keys that are seen
reach the rows that see them, whatever the kernel and the cut of its work, and no other row; turned
queries beyond fp16's range; a scale of zero."""
import pytest
import torch

import paged_bounds as PB
from paged_bounds import BF16, F16
from test_gpu_paged_bounds import attend, check

pytestmark = pytest.mark.gpu

R = pytest.importorskip("rdnattention_b200")


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    assert R.debug_read_status() == (0, 0), "a kernel recorded an expired wait"


# (kernel and cut, case)
PLANS = [
    ("few rows, whole units", dict(dtype=F16, H=8, Hkv=2, T=1, D=128, P=16, lens=[10 + i % 30 for i in range(300)])),
    ("few rows, split units", dict(dtype=BF16, H=8, Hkv=2, T=3, D=64, P=64, lens=[3000, 1000])),
    ("few rows, cluster", dict(dtype=F16, H=32, Hkv=8, T=1, D=128, P=64, lens=[700])),
    ("few rows, cluster with idle CTAs", dict(dtype=F16, H=32, Hkv=8, T=2, D=128, P=64, lens=[70])),
    ("wide heads, split units", dict(dtype=F16, H=4, Hkv=2, T=20, D=256, P=64, lens=[900, 100], kind="tree")),
    ("wide heads, whole units", dict(dtype=BF16, H=4, Hkv=2, T=20, D=160, P=16, lens=[5] * 100, kind="tree")),
    ("wide heads, cluster", dict(dtype=BF16, H=16, Hkv=8, T=4, D=256, P=16, lens=[500])),
    ("many rows, whole units", dict(dtype=F16, H=4, Hkv=2, T=20, D=128, P=16, lens=[5 + i for i in range(100)], kind="tree")),
    ("many rows, split units", dict(dtype=BF16, H=8, Hkv=2, T=40, D=64, P=64, lens=[1000, 300])),
    ("many rows, one tile", dict(dtype=F16, H=8, Hkv=8, T=24, D=128, P=64, lens=[7] * 40)),
]
IDS = [name for name, _ in PLANS]


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("kw", [kw for _, kw in PLANS], ids=IDS)
def test_a_query_row_that_is_not_finite(kw, value, rope):
    """One element of three rows (an infinity times keys of both signs gives scores of both signs, and
    their softmax is NaN): these rows are NaN, the others have the bits they have without it."""
    case = PB.plain_case(rope=rope, **kw)
    q = case["q"]
    clean = attend(**case).cpu()
    rows = {(0, 0, 0), (q.shape[0] - 1, q.shape[1] - 1, q.shape[2] - 1), (q.shape[0] // 2, 1, q.shape[2] // 2)}
    for b, h, t in rows:
        q[b, h, t, 5] = value
    got = attend(**case).cpu()
    for b, h, t in rows:
        assert torch.isnan(got[b, h, t]).all()
        got[b, h, t] = clean[b, h, t]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("slot", [0, 4])
@pytest.mark.parametrize("kw", [kw for _, kw in PLANS], ids=IDS)
def test_a_key_that_is_not_finite(kw, slot):
    """A NaN in a slot of the context that every row of one sequence and KV head sees."""
    case = PB.plain_case(**kw)
    clean = attend(**case).cpu()
    P, G = kw["P"], kw["H"] // kw["Hkv"]
    case["k_cache"][case["table"][0, slot // P], 1, slot % P, 3] = float("nan")
    got = attend(**case).cpu()
    assert torch.isnan(got[0, G:2 * G]).all()
    got[0, G:2 * G] = clean[0, G:2 * G]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("kw", [kw for _, kw in PLANS], ids=IDS)
def test_padding_rows_stay_zero_beside_nan(kw):
    """NaN in padding rows of the query (behind new_lens) and in rows outside the tables."""
    B, T = len(kw["lens"]), kw["T"]
    case = PB.plain_case(news=[T - (b % 2) * (T // 2) - int(b % 3 == 0) for b in range(B)], **kw)
    case["positions"] = torch.tensor(kw["lens"])[:, None].int() + torch.arange(T).int()
    if T > 2:
        case["positions"][:, 1] = -1
    for b, n in enumerate(case["news"]):
        case["q"][b, :, n:] = float("nan")
        if T > 2:
            case["q"][b, :, 1] = float("nan")
    got = attend(**case).cpu()
    for b, n in enumerate(case["news"]):
        assert (got[b, :, n:] == 0).all()
        if T > 2:
            assert (got[b, :, 1] == 0).all()
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("kw", [kw for _, kw in PLANS if kw["dtype"] == F16], ids=[n for n, kw in PLANS if kw["dtype"] == F16])
def test_turned_queries_beyond_fp16(kw):
    """Pairs of 6e4 turned by an eighth of a circle reach 8.5e4, beyond fp16's 65504: the turned query
    is not rounded to fp16, so the scores (times keys of 1e-3) and the output are ordinary."""
    case = PB.plain_case(**{**kw, "kind": "chain"})
    cos, sin = PB.O.tables(1, kw["D"])
    case.update(cos=cos.expand(2, -1).contiguous(), sin=sin.expand(2, -1).contiguous(),
                positions=torch.ones(len(kw["lens"]), kw["T"], dtype=torch.int32))
    case["cos"][1], case["sin"][1] = 0.5 ** 0.5, 0.5 ** 0.5
    case["q"][..., :2] = torch.tensor([6e4, 6e4])
    case["q"][..., 2:4] = torch.tensor([6e4, -6e4])
    case["k_cache"][..., :4] *= 2.0 ** -10
    check(case)


@pytest.mark.parametrize("kw", [kw for _, kw in PLANS if kw["dtype"] == BF16], ids=[n for n, kw in PLANS if kw["dtype"] == BF16])
def test_scale_of_zero(kw):
    """Products of 1e30 to 1e32 times nothing: every visible slot weighs the same."""
    case = PB.plain_case(scale=0.0, rope=False, **kw)
    case["q"] *= 1e15
    case["k_cache"] *= 1e15
    check(case)
