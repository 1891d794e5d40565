"""A cache of one page, whose page axis has any stride: the three calls give what they give with an
ordinary one."""
import pytest
import torch

pytestmark = pytest.mark.gpu

R = pytest.importorskip("rdnattention_b200")


@pytest.mark.parametrize("T,D", [(1, 128), (40, 64), (20, 256)])
@pytest.mark.parametrize("stride", [1 << 31, 1 << 40, 3])
def test_one_page(stride, T, D):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    g = torch.Generator().manual_seed(T)
    Hkv, P = 2, 300
    k, v = (torch.randn(1, Hkv, P, D, generator=g).half().cuda() for _ in range(2))
    new_k, new_v = (torch.randn(1, Hkv, T, D, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(1, 4, T, D, generator=g).half().cuda()
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    lens = torch.full((1,), 150, dtype=torch.int32, device="cuda")
    acc = torch.tensor([[T - 1]], dtype=torch.int32, device="cuda")
    outs = []
    for s0 in (k.stride(0), stride):
        kc, vc = (t.clone().as_strided(t.shape, (s0, *t.stride()[1:])) for t in (k, v))
        R.paged_kv_append(new_k, new_v, kc, vc, table, lens)
        o = R.flash_attn_paged(q, kc, vc, table, lens)
        R.paged_kv_accept(kc, vc, table, lens, acc)
        outs.append((o, kc[0].clone(), vc[0].clone()))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert R.debug_read_status() == (0, 0)
