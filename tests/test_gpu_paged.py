"""Paged KV-cache operators on the GPU against their 64-bit definitions
(paged_oracle.py, which derives the bounds): lengths from zero up, ragged padded
batches, trees, windows, page sizes, strides, stale values behind the end, bad
page table entries, streams, captured steps, and a run of the three together."""
import pytest
import torch

import paged_oracle as O

pytestmark = pytest.mark.gpu

R = pytest.importorskip("rdnattention_b200")


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    assert R.debug_read_status() == (0, 0), "a kernel recorded an expired wait"


F16, BF16 = torch.float16, torch.bfloat16


def make_cache(g, dtype, lens, T, Hkv, P, D, spare=2, order="phsd"):
    """(k_cache, v_cache, table): every sequence has room for T more tokens; pages in random order."""
    need = [max(1, -(-(max(n, 0) + T) // P)) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=g).int()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n

    def cache():
        if order == "phsd":
            return torch.randn(total, Hkv, P, D, generator=g).to(dtype)
        return torch.randn(total, P, Hkv, D, generator=g).to(dtype).transpose(1, 2)

    return cache(), cache(), table


def tree(g, B, T):
    """Random trees: (mask [B, T, T], depth [B, T])."""
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    depth = torch.zeros(B, T, dtype=torch.int64)
    for b in range(B):
        for t in range(T):
            if t:
                par = int(torch.randint(max(0, t - 5), t, (1,), generator=g))
                mask[b, t] = mask[b, par]
                depth[b, t] = depth[b, par] + 1
            mask[b, t, t] = True
    return mask, depth


def cuda(*ts):
    """To the GPU with the strides kept."""
    out = []
    for t in ts:
        if t is None or t.is_cuda:
            out.append(t)
            continue
        d = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
        out.append(d.copy_(t))
    return out if len(out) > 1 else out[0]


def check(got, ref, bound):
    err = (got.double().cpu() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside; worst {(err / bound).max().item():.3g} bounds"


def attend(q, kc, vc, table, lens, news=None, mask=None, positions=None, cos=None, sin=None, **kw):
    a = cuda(q, kc, vc, table)
    return R.flash_attn_paged(*a, cuda(torch.tensor(lens, dtype=torch.int32)),
                              new_lens=None if news is None else cuda(torch.tensor(news, dtype=torch.int32)),
                              tree_mask=cuda(mask), positions=cuda(positions), rot_cos=cuda(cos), rot_sin=cuda(sin),
                              **kw)


def run_case(dtype, H, Hkv, T, D, P, lens, news=None, kind="chain", window=-1, rope=True, order="phsd", seed=0):
    g = torch.Generator().manual_seed(seed + 17 * T + D + P)
    B = len(lens)
    kc, vc, table = make_cache(g, dtype, lens, T, Hkv, P, D, order=order)
    q = (2 * torch.randn(B, H, T, D, generator=g)).to(dtype)
    mask = positions = cos = sin = None
    if kind == "tree":
        mask, depth = tree(g, B, T)
        positions = (torch.tensor(lens)[:, None].clamp(min=0) + depth).int()
    if rope:
        cos, sin = O.tables(max(lens) + T + 1, D)
    got = attend(q, kc, vc, table, lens, news, mask, positions, cos, sin, window_size=window)
    ref, bound = O.attention(q, kc, vc, table, lens, news, mask, positions, cos, sin, window)
    check(got, ref, bound)
    return got


CASES = [
    # one token: lengths 0, 1, tile edges
    dict(dtype=F16, H=8, Hkv=2, T=1, D=128, P=64, lens=[0, 1, 30, 31, 32, 63, 64, 65, 700]),
    dict(dtype=BF16, H=8, Hkv=8, T=1, D=64, P=16, lens=[5, 0, 1000, 333]),
    dict(dtype=F16, H=16, Hkv=1, T=1, D=128, P=32, lens=[4097]),
    dict(dtype=BF16, H=5, Hkv=1, T=1, D=256, P=64, lens=[900, 0, 64]),
    # every head_dim
    *[dict(dtype=dt, H=4, Hkv=2, T=3, D=D, P=16, lens=[100, 37], kind="tree")
      for D in (32, 64, 96, 128, 160, 192, 224, 256) for dt in (F16, BF16)],
    # page sizes: smaller than a tile, larger, ending inside a tile, one page
    *[dict(dtype=F16, H=6, Hkv=2, T=5, D=64, P=P, lens=[P - 1, P, 3 * P + 7, 0, 500])
      for P in (8, 16, 32, 64, 72, 100, 128, 777)],
    # ragged padded batch, some sequences without new tokens
    dict(dtype=F16, H=8, Hkv=2, T=7, D=128, P=16, lens=[50, 0, 0, 300, 17], news=[7, 0, 3, 1, 5]),
    dict(dtype=BF16, H=12, Hkv=3, T=13, D=96, P=16, lens=[500, 0, 123], news=[13, 2, 9], kind="tree", window=100),
    # many rows: row tiles, several tokens across them
    dict(dtype=F16, H=8, Hkv=2, T=64, D=128, P=64, lens=[1000, 3], kind="tree"),
    dict(dtype=BF16, H=32, Hkv=8, T=64, D=128, P=16, lens=[200, 0], news=[64, 33], kind="tree"),
    dict(dtype=F16, H=8, Hkv=1, T=33, D=64, P=16, lens=[257], kind="tree"),
    dict(dtype=F16, H=3, Hkv=1, T=150, D=64, P=32, lens=[10], kind="tree", window=4),
    dict(dtype=F16, H=2, Hkv=2, T=256, D=32, P=16, lens=[77], kind="tree"),
    dict(dtype=F16, H=4, Hkv=2, T=300, D=128, P=64, lens=[0, 513]),
    dict(dtype=BF16, H=7, Hkv=1, T=130, D=160, P=72, lens=[90, 1], news=[130, 127]),
    # windows: inside one tile, over tiles, longer than the context
    *[dict(dtype=F16, H=8, Hkv=2, T=T, D=128, P=16, lens=[400, 3, 0], kind=kind, window=w)
      for T in (1, 20) for kind in ("chain", "tree") for w in (1, 2, 33, 200, 5000)],
    # no rotation, other cache order
    dict(dtype=F16, H=8, Hkv=4, T=4, D=128, P=16, lens=[333, 20], rope=False, order="pshd"),
    dict(dtype=BF16, H=16, Hkv=4, T=40, D=64, P=64, lens=[333, 20], kind="tree", order="pshd"),
    # long: split over many CTAs
    dict(dtype=F16, H=8, Hkv=2, T=1, D=128, P=64, lens=[20011]),
    dict(dtype=BF16, H=8, Hkv=2, T=16, D=128, P=16, lens=[9001, 13], kind="tree"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c.values()))
def test_attention(case):
    run_case(**case)


@pytest.mark.parametrize("T,kind,window", [(1, "chain", -1), (4, "chain", 70), (5, "tree", -1), (16, "tree", 90),
                                           (64, "tree", -1), (40, "chain", -1)])
@pytest.mark.parametrize("length", [0, 1, 64, 700, 6001])
@pytest.mark.parametrize("dtype,H,Hkv,D,P", [(F16, 32, 8, 128, 64), (BF16, 24, 12, 64, 16), (F16, 8, 8, 256, 72)])
def test_single_sequence(T, kind, window, length, dtype, H, Hkv, D, P):
    """One sequence with enough heads for the cluster form, from fewer key tiles than CTAs to many."""
    run_case(dtype, H, Hkv, T, D, P, [length], kind=kind, window=window)


def test_single_sequence_with_nothing_to_see():
    """No key, no new token, masks that hide everything, NaN in the cache: zeros."""
    g = torch.Generator().manual_seed(21)
    for T, D in ((1, 128), (8, 128), (8, 256)):
        kc, vc, table = make_cache(g, F16, [0], T, 8, 16, D)
        kc.fill_(float("nan"))
        vc.fill_(float("nan"))
        q = torch.randn(1, 32, T, D, generator=g).to(F16)
        assert (attend(q, kc, vc, table, [0], [0]) == 0).all()
        assert (attend(q, kc, vc, table, [50], [0]) == 0).all()
        vc.zero_()
        kc.zero_()
        assert (attend(q, kc, vc, table, [0], mask=torch.zeros(T, T, dtype=torch.bool)) == 0).all()


def test_masks_that_leave_rows_empty():
    """Rows whose mask is all false see the context alone; over an empty context they are zero."""
    g = torch.Generator().manual_seed(3)
    B, H, Hkv, T, D, P = 3, 4, 2, 40, 64, 16
    lens = [0, 70, 0]
    kc, vc, table = make_cache(g, F16, lens, T, Hkv, P, D)
    q = torch.randn(B, H, T, D, generator=g).to(F16)
    mask = torch.rand(B, T, T, generator=g) < 0.1
    mask[:, 3] = False
    mask[2] = False
    got = attend(q, kc, vc, table, lens, mask=mask)
    ref, bound = O.attention(q, kc, vc, table, lens, mask=mask)
    check(got, ref, bound)
    assert (got[0, :, 3] == 0).all() and (got[2] == 0).all()
    # one mask for the whole batch, as [T, T] and [1, T, T], and as a strided view
    wide = torch.zeros(T, 2 * T, dtype=torch.bool)
    wide[:, :T] = mask[0]
    ref, bound = O.attention(q, kc, vc, table, lens, mask=mask[:1].expand(B, T, T))
    for m in (mask[0], mask[:1], wide[:, :T]):
        check(attend(q, kc, vc, table, lens, mask=m), ref, bound)


@pytest.mark.parametrize("T,H,kind", [(1, 8, "chain"), (9, 8, "tree"), (70, 4, "tree")])
@pytest.mark.parametrize("P", [16, 64, 100])
def test_stale_slots_may_hold_anything(T, H, kind, P):
    """NaN and infinities behind the new tokens, in unused pages, behind new_lens and before the
    window do not reach the output."""
    g = torch.Generator().manual_seed(4)
    lens, news, window = [130, 64, 31], [T, max(T - 2, 1), 1], 40
    kc, vc, table = make_cache(g, F16, lens, T, 2, P, 64)
    q = torch.randn(3, H, T, 64, generator=g).to(F16)
    mask = tree(g, 3, T)[0] if kind == "tree" else None
    ref, bound = O.attention(q, kc, vc, table, lens, news, mask, window=window)
    used = torch.zeros(kc.shape[0], P, dtype=torch.bool)
    for b in range(3):
        first = max(0, lens[b] - window) if kind == "tree" else max(0, lens[b] + 1 - window)
        for s in range(first, lens[b] + news[b]):
            used[table[b, s // P], s % P] = True
    for c, x in ((kc, float("nan")), (vc, float("inf"))):
        c.masked_fill_(~used[:, None, :, None], x)
    check(attend(q, kc, vc, table, lens, news, mask, window_size=window), ref, bound)


def test_bad_pages_read_as_zeros_and_bad_lengths_are_clamped():
    g = torch.Generator().manual_seed(5)
    lens = [200, 100, 60]
    kc, vc, table = make_cache(g, F16, lens, 4, 2, 16, 64)
    table[0, 3], table[0, 5], table[1, 2] = -7, 2 ** 31 - 1, kc.shape[0]
    q = torch.randn(3, 4, 4, 64, generator=g).to(F16)
    check(attend(q, kc, vc, table, lens), *O.attention(q, kc, vc, table, lens))
    lens = [-5, 2 ** 31 - 1, 60]
    check(attend(q, kc, vc, table, lens, [9, 4, -1]), *O.attention(q, kc, vc, table, lens, [9, 4, -1]))


def test_positions_outside_the_tables_give_zero_rows():
    g = torch.Generator().manual_seed(6)
    lens = [50, 20]
    kc, vc, table = make_cache(g, BF16, lens, 5, 2, 16, 128)
    q = torch.randn(2, 4, 5, 128, generator=g).to(BF16)
    cos, sin = O.tables(60, 128)
    pos = torch.tensor([[50, 60, 3, -1, 59], [0, 1, 2, 2 ** 31 - 1, 4]], dtype=torch.int32)
    got = attend(q, kc, vc, table, lens, positions=pos, cos=cos, sin=sin)
    check(got, *O.attention(q, kc, vc, table, lens, positions=pos, cos=cos, sin=sin))
    assert (got[0, :, 1] == 0).all() and (got[0, :, 3] == 0).all() and (got[1, :, 3] == 0).all()


def test_strided_query_and_output_and_scale():
    g = torch.Generator().manual_seed(7)
    B, H, Hkv, T, D = 2, 8, 2, 6, 64
    lens = [99, 300]
    kc, vc, table = make_cache(g, F16, lens, T, Hkv, 16, D)
    q = torch.randn(B, T, H, D, generator=g).to(F16).transpose(1, 2)
    buf = torch.full((B, T, H, 2 * D), 7.0, dtype=F16, device="cuda")
    out = buf[..., :D].transpose(1, 2)
    got = attend(q, kc, vc, table, lens, scale=-0.3, out=out)
    assert got is out and (buf[..., D:] == 7).all()
    check(got, *O.attention(q, kc, vc, table, lens, scale=-0.3))
    wide = torch.zeros(B, table.shape[1] + 5, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    check(attend(q, kc, vc, wide[:, :table.shape[1]], lens), *O.attention(q, kc, vc, table, lens))


def test_contiguous_cache_is_one_page_per_sequence():
    """[B, Hkv, S, D] as a cache of B pages; the chain equals the causal strided call."""
    g = torch.Generator().manual_seed(8)
    B, H, Hkv, S, D, T = 3, 8, 2, 501, 128, 3
    k, v = (torch.randn(B, Hkv, S, D, generator=g).to(F16).cuda() for _ in range(2))
    q = torch.randn(B, H, T, D, generator=g).to(F16).cuda()
    table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
    lens = torch.full((B,), S - T, dtype=torch.int32, device="cuda")
    a = R.flash_attn_paged(q, k, v, table, lens)
    b = R.flash_attn_strided(q, k, v, is_causal=True)
    assert (a.float() - b.float()).abs().max().item() < 2e-3


def test_more_sequences_than_one_launch():
    """2100 sequences: two launches that share the workspace."""
    lens = [(i * 7) % 50 for i in range(2100)]
    run_case(F16, 2, 1, 2, 32, 16, lens, rope=False)


def test_results_do_not_depend_on_timing():
    a = run_case(F16, 32, 8, 16, 128, 16, [8000, 500, 3], kind="tree")
    b = run_case(F16, 32, 8, 16, 128, 16, [8000, 500, 3], kind="tree")
    assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """Pages more than 2^32 bytes into the cache."""
    n, P, Hkv, D = 2 ** 32 // (64 * 2 * 128 * 2) + 300, 64, 2, 128
    kc, vc = (torch.zeros(n, Hkv, P, D, dtype=F16, device="cuda") for _ in range(2))
    assert kc.numel() * 2 > 2 ** 32
    g = torch.Generator().manual_seed(9)
    pages = torch.tensor([[n - 1, 0, n - 7, 5, n - 100]], dtype=torch.int32)
    lens, T = torch.tensor([200], dtype=torch.int32), 70
    key, value = (torch.randn(1, Hkv, 320, D, generator=g).to(F16) for _ in range(2))
    small_k, small_v = (torch.zeros(5, Hkv, P, D, dtype=F16) for _ in range(2))
    small = torch.arange(5, dtype=torch.int32)[None]
    zero = torch.zeros(1, dtype=torch.int32)
    R.paged_kv_append(*cuda(key, value), kc, vc, *cuda(pages, zero))
    K, _, V = O.append(key, value, small_k, small_v, small, zero)
    for i, pg in enumerate(pages[0].tolist()):
        assert torch.equal(kc[pg].cpu().double(), K[i]) and torch.equal(vc[pg].cpu(), V[i])
    q = torch.randn(1, 4, T, D, generator=g).to(F16)
    got = R.flash_attn_paged(q.cuda(), kc, vc, pages.cuda(), lens.cuda())
    check(got, *O.attention(q, K.to(F16), V, small, lens))
    acc = torch.tensor([[60, 3]], dtype=torch.int32)
    R.paged_kv_accept(kc, vc, pages.cuda(), lens.cuda(), acc.cuda())
    K2, V2 = O.accept(K.to(F16), V, small, lens, acc)
    for i, pg in enumerate(pages[0].tolist()):
        assert torch.equal(kc[pg].cpu(), K2[i]) and torch.equal(vc[pg].cpu(), V2[i])


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Hkv,T,D,P,lens,news,rope,order", [
    (1, 8, 1, 128, 64, [100], None, True, "phsd"),
    (3, 2, 1, 64, 16, [0, 15, 16], None, True, "pshd"),
    (4, 3, 61, 96, 16, [5, 0, 77, 31], [61, 0, 9, 60], True, "phsd"),
    (2, 1, 300, 256, 72, [70, 3], [300, 299], True, "phsd"),
    (2, 5, 7, 32, 8, [7, 8], None, False, "phsd"),
    (1, 2, 1000, 160, 100, [50], None, True, "pshd"),
])
def test_append(dtype, B, Hkv, T, D, P, lens, news, rope, order):
    g = torch.Generator().manual_seed(T + D)
    kc, vc, table = make_cache(g, dtype, lens, T, Hkv, P, D, order=order)
    key = torch.randn(B, T, Hkv, D, generator=g).to(dtype).transpose(1, 2)
    value = torch.randn(B, Hkv, T, D, generator=g).to(dtype)
    cos, sin = O.tables(max(lens) + T, D) if rope else (None, None)
    pos = torch.randint(0, max(lens) + T, (B, T), generator=g).int() if T % 2 else None
    L = torch.tensor(lens, dtype=torch.int32)
    N = None if news is None else torch.tensor(news, dtype=torch.int32)
    K, bound, V = O.append(key, value, kc, vc, table, lens, news, pos, cos, sin)
    dk, dv = cuda(kc, vc)
    out = R.paged_kv_append(*cuda(key, value), dk, dv, *cuda(table, L), new_lens=cuda(N), positions=cuda(pos),
                            rot_cos=cuda(cos), rot_sin=cuda(sin))
    assert out[0] is dk and out[1] is dv
    check(dk, K, bound)  # bound 0 outside the new rows: left bit for bit
    assert torch.equal(dv.cpu(), V)


def test_append_skips_what_it_cannot_place():
    """Bad pages, positions outside the tables, slots behind the table: not written, nothing else touched."""
    g = torch.Generator().manual_seed(11)
    B, Hkv, T, D, P = 4, 2, 20, 64, 16
    kc, vc, table = make_cache(g, F16, [30] * B, T, Hkv, P, D)
    table[0, 2], table[1, 3], table[2, 2] = -1, kc.shape[0], -2 ** 31
    lens, news = [30, 40, 2 ** 31 - 1, -9], [20, 20, 20, 99]
    cos, sin = O.tables(50, D)
    pos = torch.randint(-3, 60, (B, T), generator=g).int()
    key, value = (torch.randn(B, Hkv, T, D, generator=g).to(F16) for _ in range(2))
    K, bound, V = O.append(key, value, kc, vc, table, lens, news, pos, cos, sin)
    dk, dv = cuda(kc, vc)
    R.paged_kv_append(*cuda(key, value), dk, dv, *cuda(table, torch.tensor(lens, dtype=torch.int32)),
                      new_lens=cuda(torch.tensor(news, dtype=torch.int32)), positions=cuda(pos), rot_cos=cuda(cos),
                      rot_sin=cuda(sin))
    check(dk, K, bound)
    assert torch.equal(dv.cpu(), V)


# ------------------------------------------------------------------- accept
@pytest.mark.parametrize("dtype,Hkv,D,P,A,order", [(F16, 8, 128, 64, 4, "phsd"), (BF16, 3, 96, 16, 17, "pshd"),
                                                   (F16, 1, 32, 8, 100, "phsd"), (BF16, 2, 256, 72, 256, "phsd"),
                                                   (F16, 2, 64, 16, 1, "phsd")])
def test_accept(dtype, Hkv, D, P, A, order):
    """Any indices: ascending paths, swaps, the same token twice, entries to skip."""
    g = torch.Generator().manual_seed(A)
    lens = [100, 0, 33, 7]
    kc, vc, table = make_cache(g, dtype, lens, 260, Hkv, P, D, order=order)
    acc = torch.randint(-2, 260, (4, A), generator=g).int()
    acc[0] = torch.randperm(260, generator=g)[:A].sort().values.int()
    acc[1] = torch.arange(A - 1, -1, -1).int()
    table[3, 0] = -1
    n = torch.tensor([A, A, max(A - 1, 0), 999], dtype=torch.int32)
    L = torch.tensor(lens, dtype=torch.int32)
    for nn in (n, None):
        K, V = O.accept(kc, vc, table, lens, acc, nn)
        dk, dv = cuda(kc, vc)
        R.paged_kv_accept(dk, dv, *cuda(table, L, acc), accepted_lens=cuda(nn))
        assert torch.equal(dk.cpu(), K) and torch.equal(dv.cpu(), V)


# ------------------------------------------------------------- runs of them
def _step(key, value, q, kc, vc, table, lens, mask, pos, cos, sin, acc, n):
    R.paged_kv_append(key, value, kc, vc, table, lens, positions=pos, rot_cos=cos, rot_sin=sin)
    o = R.flash_attn_paged(q, kc, vc, table, lens, tree_mask=mask, positions=pos, rot_cos=cos, rot_sin=sin)
    R.paged_kv_accept(kc, vc, table, lens, acc, accepted_lens=n)
    lens += n
    return o


def _speculative_inputs(seed, B=3, H=8, Hkv=2, T=12, D=64, P=16, steps=4):
    g = torch.Generator().manual_seed(seed)
    lens = [40, 0, 15]
    kc, vc, table = make_cache(g, F16, [n + T * steps for n in lens], T, Hkv, P, D)
    cos, sin = O.tables(400, D)
    turns = []
    for _ in range(steps):
        mask, depth = tree(g, B, T)
        path = torch.zeros(B, 4, dtype=torch.int32)
        n = torch.zeros(B, dtype=torch.int32)
        for b in range(B):
            leaf = int(torch.randint(0, T, (1,), generator=g))
            line = mask[b, leaf].nonzero().flatten()[:4]
            path[b, :len(line)] = line.int()
            n[b] = len(line)
        turns.append((torch.randn(B, Hkv, T, D, generator=g).to(F16), torch.randn(B, Hkv, T, D, generator=g).to(F16),
                      torch.randn(B, H, T, D, generator=g).to(F16), mask, depth, path, n))
    return lens, kc, vc, table, cos, sin, turns


def _speculative_oracle(lens, kc, vc, table, cos, sin, turns):
    L, outs = torch.tensor(lens), []
    for key, value, q, mask, depth, path, n in turns:
        pos = (L[:, None] + depth).int()
        K, _, vc = O.append(key, value, kc, vc, table, L.tolist(), None, pos, cos, sin)
        kc = K.to(F16)
        outs.append(O.attention(q, kc, vc, table, L.tolist(), None, mask, pos, cos, sin))
        kc, vc = O.accept(kc, vc, table, L.tolist(), path, n)
        L = L + n
    return outs, L


def test_speculative_steps_together():
    """Append, attend, accept, four times.  The kernel turns keys in 32 bits and the oracle in 64, so a key
    may round to the neighbour, 2 u away: the scores then move by 3 d instead of d, hence 3 bounds."""
    lens, kc, vc, table, cos, sin, turns = _speculative_inputs(1)
    want, L = _speculative_oracle(lens, kc, vc, table, cos, sin, turns)
    dk, dv, dt, dc, ds = cuda(kc, vc, table, cos, sin)
    dl = torch.tensor(lens, dtype=torch.int32).cuda()
    for (key, value, q, mask, depth, path, n), (ref, bound) in zip(turns, want):
        pos = (dl[:, None] + depth.cuda()).int()
        o = _step(*cuda(key, value, q), dk, dv, dt, dl, mask.cuda(), pos, dc, ds, *cuda(path, n))
        check(o, ref, 3 * bound)
    assert torch.equal(dl.cpu().long(), L)


def test_captured_step_replays_with_new_lengths():
    """One captured step, replayed with other inputs, lengths and trees."""
    lens, kc, vc, table, cos, sin, turns = _speculative_inputs(2)
    want, L = _speculative_oracle(lens, kc, vc, table, cos, sin, turns)
    dk, dv, dt, dc, ds = cuda(kc, vc, table, cos, sin)
    dl = torch.tensor(lens, dtype=torch.int32).cuda()
    buf = [t.cuda() for t in turns[0]]
    key, value, q, mask, depth, path, n = buf

    def step():
        pos = (dl[:, None] + depth).int()
        return _step(key, value, q, dk, dv, dt, dl, mask, pos, dc, ds, path, n)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # warm-up changes the cache: put it back
    torch.cuda.current_stream().wait_stream(side)
    dk.copy_(kc)
    dv.copy_(vc)
    dl.copy_(torch.tensor(lens, dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn, (ref, bound) in zip(turns, want):
        for dst, src in zip(buf, turn):
            dst.copy_(src)
        graph.replay()
        check(out, ref, 3 * bound)
    assert torch.equal(dl.cpu().long(), L)


@pytest.mark.parametrize("T,kind", [(1, "chain"), (20, "tree")])
def test_captured_single_sequence(T, kind):
    """The forms a single sequence takes, captured, replayed over growing lengths, two replays in a row."""
    g = torch.Generator().manual_seed(31)
    H, Hkv, D, P = 32, 8, 128, 16
    kc, vc, table = make_cache(g, BF16, [900], T, Hkv, P, D)
    q = torch.randn(1, H, T, D, generator=g).to(BF16)
    mask = tree(g, 1, T)[0] if kind == "tree" else None
    dq, dk, dv, dt, dm = cuda(q), *cuda(kc, vc, table), cuda(mask)
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    R.flash_attn_paged(dq, dk, dv, dt, lens, tree_mask=dm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [R.flash_attn_paged(dq, dk, dv, dt, lens, tree_mask=dm) for _ in range(2)]
    for n in (0, 5, 64, 333, 900):
        lens.fill_(n)
        graph.replay()
        graph.replay()
        ref, bound = O.attention(q, kc, vc, table, [n], mask=mask)
        for out in outs:
            check(out, ref, bound)


@pytest.mark.parametrize("dtype,H,D,P,T", [(F16, 2, 64, 16, 6), (BF16, 4, 128, 8, 5), (F16, 4, 256, 64, 6),
                                           (BF16, 4, 128, 16, 40), (F16, 2, 64, 64, 150)])
def test_slots_no_token_sees_in_front_of_a_tree_window(dtype, H, D, P, T):
    """Every token of a tree sees itself, so the context's part of a window of w is w - 1 at most:
    slot len - w may be stale."""
    g = torch.Generator().manual_seed(D + T)
    lens, w = [37, 130], 20
    kc, vc, table = make_cache(g, dtype, lens, T, 2, P, D)
    q = torch.randn(2, H, T, D, generator=g).to(dtype)
    mask, _ = tree(g, 2, T)
    ref, bound = O.attention(q, kc, vc, table, lens, mask=mask, window=w)
    for b, n in enumerate(lens):
        for s in range(n - w + 1):
            kc[table[b, s // P], :, s % P] = float("nan")
            vc[table[b, s // P], :, s % P] = float("inf")
    check(attend(q, kc, vc, table, lens, mask=mask, window_size=w), ref, bound)


def test_python_refusals():
    """What the entry points refuse before a launch."""
    dev = "cuda"
    kc = torch.zeros(4, 2, 16, 64, dtype=F16, device=dev)
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    q, kv = (torch.zeros(2, h, 3, 64, dtype=F16, device=dev) for h in (4, 2))

    def attend(q=q, k=kc, v=kc, t=table, n=lens, **kw):
        return R.flash_attn_paged(q, k, v, t, n, **kw)

    mask = torch.ones(3, 3, dtype=torch.bool, device=dev)
    cos = torch.zeros(10, 32, device=dev)
    i32 = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    for call, match in [
        (lambda: attend(k=kc.float(), v=kc.float()), "float16 or bfloat16"),
        (lambda: attend(v=kc.bfloat16()), "v_cache must be torch.float16"),
        (lambda: attend(v=kc[:3]), "v_cache must have shape"),
        (lambda: attend(k=kc[0], v=kc[0]), "k_cache must be 4D"),
        (lambda: attend(k=kc.transpose(2, 3), v=kc.transpose(2, 3)), "contiguous head_dim"),
        (lambda: attend(t=table.long()), "page_table must be torch.int32"),
        (lambda: attend(t=table[0]), "page_table must be 2D"),
        (lambda: attend(t=table.cpu()), "same device"),
        (lambda: attend(n=lens[:1]), "cache_lens must have shape"),
        (lambda: attend(n=torch.zeros(4, dtype=torch.int32, device=dev)[::2]), "cache_lens must be contiguous"),
        (lambda: attend(q=q.bfloat16()), "query must be torch.float16"),
        (lambda: attend(q=q[:1]), "query must be 4D"),
        (lambda: attend(q=q[:, :3]), "multiple of the cache's heads"),
        (lambda: attend(q=q.transpose(2, 3).contiguous().transpose(2, 3)), "query must have a contiguous head_dim"),
        (lambda: attend(new_lens=lens.float()), "new_lens must be torch.int32"),
        (lambda: attend(positions=i32.t().contiguous().t()), "positions must be contiguous"),
        (lambda: attend(positions=i32[:, :2]), "positions must have shape"),
        (lambda: attend(tree_mask=mask.int()), "tree_mask must be torch.bool"),
        (lambda: attend(tree_mask=mask[:2]), "tree_mask must be"),
        (lambda: attend(tree_mask=mask.t()[:, :].t()[:, torch.tensor([2, 1, 0], device=dev)].t()), "contiguous rows"),
        (lambda: attend(rot_cos=cos), "both rot_cos and rot_sin"),
        (lambda: attend(rot_cos=cos, rot_sin=cos[:5]), "shapes must match"),
        (lambda: attend(rot_cos=cos[:, :16].contiguous(), rot_sin=cos[:, :16].contiguous()), "head_dim // 2"),
        (lambda: attend(out=torch.zeros_like(q).bfloat16()), "out must be torch.float16"),
        (lambda: attend(out=torch.zeros_like(kv)), "out must have shape"),
        (lambda: attend(out=q), "must not share memory"),
        (lambda: attend(rot_cos=cos[:0], rot_sin=cos[:0]), "no rows"),
        (lambda: R.paged_kv_append(q, kv, kc, kc, table, lens), "key must be 4D"),
        (lambda: R.paged_kv_append(kv, kv[:, :, :2], kc, kc, table, lens), "key and value shapes"),
        (lambda: R.paged_kv_accept(kc, kc, table, lens, i32.float()), "accepted must be torch.int32"),
        (lambda: R.paged_kv_accept(kc, kc, table, lens, i32[:1]), "accepted must be contiguous"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(R.RDNAttentionError, match="head_dim 48"):
        x = torch.zeros(4, 2, 16, 48, dtype=F16, device=dev)
        attend(k=x, v=x)
    with pytest.raises(R.RDNAttentionError, match="page_size"):
        x = torch.zeros(4, 2, 12, 64, dtype=F16, device=dev)
        attend(k=x, v=x)
    big = torch.zeros(2, 4, 257, 64, dtype=F16, device=dev)
    with pytest.raises(ValueError, match="at most 256"):
        attend(q=big, tree_mask=torch.ones(257, 257, dtype=torch.bool, device=dev))
    with pytest.raises(ValueError, match="at most 256"):
        R.paged_kv_accept(kc, kc, table, lens, torch.zeros(2, 257, dtype=torch.int32, device=dev))
    # nothing to do is not an error
    empty = torch.zeros(2, 4, 0, 64, dtype=F16, device=dev)
    assert attend(q=empty).shape == empty.shape
    assert R.paged_kv_accept(kc, kc, table, lens, i32[:, :0].contiguous())[0] is kc


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    g = torch.Generator().manual_seed(13)
    data = []
    for s in range(2):
        lens = [6000 + 100 * s]
        kc, vc, table = make_cache(g, F16, lens, 8, 2, 64, 128)
        q = torch.randn(1, 8, 8, 128, generator=g).to(F16)
        data.append((cuda(q, kc, vc, table) + [cuda(torch.tensor(lens, dtype=torch.int32))],
                     O.attention(q, kc, vc, table, lens)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(R.flash_attn_paged(*data[i][0]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            check(o, *data[i][1])
