"""Paged KV-cache operators without a GPU: what the C ABI and the Python entry
points refuse before they touch a device, the workspace's size, and the oracle
against a dense computation."""
import struct
import subprocess
from pathlib import Path

import pytest
import torch

import paged_oracle as O
import rdnattention_b200 as R
from rdnattention_b200 import paged

CS = (8 * 64 * 128, 64 * 128, 128)  # page / head / slot strides of a [pages, 8, 64, 128] cache


def _message(rc):
    return rc, R._lib_handle().rdna_get_error().decode()


def _pack(layout, *values):
    """The struct's bytes; values beyond a field's range are the caller's mistake, None is a null pointer."""
    return layout.pack(*(0 if v is None else v for v in values))


def _cache(a):
    return (a["kc"], a["vc"], a["table"], a["lens"], *a["kcs"], *a["vcs"], a["ts"], a["B"], a["Hkv"], a["D"],
            a["pages"], a["P"], a["mp"], a["dt"], 0)


def _append(**kw):
    a = dict(key=16, value=16, kc=16, vc=16, table=16, lens=16, news=None, pos=None, cos=None, sin=None, ks=CS, vs=CS,
             kcs=CS, vcs=CS, ts=4, B=2, Hkv=8, T=3, D=128, pages=8, P=64, mp=4, rows=0, dt=0)
    a.update(kw)
    return _message(R._lib_handle().rdna_paged_kv_append(
        _pack(paged._APPEND, *_cache(a), a["key"], a["value"], a["news"], a["pos"], a["cos"], a["sin"], *a["ks"],
              *a["vs"], a["T"], a["rows"]), None))


def _attend(**kw):
    a = dict(q=16, kc=16, vc=16, o=16, table=16, lens=16, news=None, mask=None, pos=None, cos=None, sin=None, qs=CS,
             kcs=CS, vcs=CS, os=CS, mb=0, mt=0, ts=4, B=2, H=8, Hkv=8, T=3, D=128, pages=8, P=64, mp=4, rows=0,
             scale=0.1, window=-1, dt=0, ws=256, wsb=1 << 40)
    a.update(kw)
    return _message(R._lib_handle().rdna_attention_forward_paged(
        _pack(paged._ATTENTION, *_cache(a), a["q"], a["o"], a["news"], a["mask"], a["pos"], a["cos"], a["sin"],
              a["ws"], a["wsb"], *a["qs"], *a["os"], a["mb"], a["mt"], a["H"], a["T"], a["rows"], a["window"],
              a["scale"], 0), None))


def _accept(**kw):
    a = dict(kc=16, vc=16, table=16, lens=16, acc=16, al=None, kcs=CS, vcs=CS, ts=4, B=2, Hkv=8, D=128, pages=8, P=64,
             mp=4, A=4, dt=0)
    a.update(kw)
    return _message(R._lib_handle().rdna_paged_kv_accept(
        _pack(paged._ACCEPT, *_cache(a), a["acc"], a["al"], a["A"], 0), None))


COMMON = [
    (dict(kc=None), "null tensor pointer"), (dict(vc=None), "null tensor pointer"),
    (dict(table=None), "null tensor pointer"), (dict(lens=None), "null tensor pointer"),
    (dict(dt=2), "dtype must be"), (dict(dt=-1), "dtype must be"),
    (dict(B=0), "empty problem"), (dict(Hkv=0), "empty problem"), (dict(pages=0), "empty problem"),
    (dict(mp=0), "empty problem"), (dict(D=48), "unsupported head_dim"), (dict(D=288), "unsupported head_dim"),
    (dict(D=0), "unsupported head_dim"), (dict(P=0), "unsupported page_size"), (dict(P=4), "unsupported page_size"),
    (dict(P=48), "unsupported page_size"), (dict(mp=1 << 25), "exceeds 2^30"), (dict(kc=24), "16-byte aligned"),
    (dict(table=18), "4-byte aligned"), (dict(lens=17), "4-byte aligned"), (dict(ts=-4), "strides must be positive"),
    (dict(kcs=(CS[0], 0, 128)), "strides must be positive"), (dict(vcs=(CS[0], CS[1], 132)), "multiples of 16 bytes"),
    (dict(kcs=(1 << 40, CS[1], 128)), "stride too large"), (dict(pages=1 << 31), "too many pages"),
]


@pytest.mark.parametrize("call", [_append, _attend, _accept])
@pytest.mark.parametrize("kw,needle", COMMON)
def test_cache_refusals(call, kw, needle):
    rc, msg = call(**kw)
    assert rc == -3 and needle in msg, msg


ROPE = [(dict(cos=16), "both rot_cos and rot_sin"), (dict(sin=16), "both rot_cos and rot_sin"),
        (dict(cos=20, sin=32, rows=4), "16-byte aligned"), (dict(cos=16, sin=32, rows=1 << 31), "too many rotation"),
        (dict(pos=18), "4-byte aligned"), (dict(news=18), "4-byte aligned")]


@pytest.mark.parametrize("kw,needle", ROPE + [
    (dict(key=None), "null tensor pointer"), (dict(value=8), "16-byte aligned"),
    (dict(ks=(CS[0], -128, 128)), "strides must be positive"), (dict(vs=(CS[0], CS[1], 4)), "multiples of 16 bytes"),
    (dict(T=(1 << 30) + 1), "sequence too long"), (dict(B=1 << 24, T=1 << 30), "too large for one launch")])
def test_append_refusals(kw, needle):
    rc, msg = _append(**kw)
    assert rc == -3 and needle in msg and msg.startswith("Paged cache append failed: "), msg


@pytest.mark.parametrize("kw,needle", ROPE + [
    (dict(q=None), "null tensor pointer"), (dict(o=None), "null tensor pointer"), (dict(q=8), "16-byte aligned"),
    (dict(H=12), "positive multiple"), (dict(H=0), "positive multiple"), (dict(mask=16, T=257), "more than 256"),
    (dict(mask=16, mt=-1), "strides must be positive"), (dict(T=1 << 29), "sequence too long"),
    (dict(qs=(0, CS[1], 128)), "strides must be positive"), (dict(os=(CS[0], CS[1], 60)), "multiples of 16 bytes"),
    (dict(ws=None), "workspace missing"), (dict(wsb=100), "workspace missing"), (dict(ws=128), "256-byte aligned"),
    (dict(T=1 << 24, mp=1 << 24), "too large for one launch")])
def test_attention_refusals(kw, needle):
    rc, msg = _attend(**kw)
    assert rc == -3 and needle in msg and msg.startswith("Attention (paged) failed: "), msg


@pytest.mark.parametrize("kw,needle", [
    (dict(acc=None), "null tensor pointer"), (dict(A=257), "more than 256"), (dict(acc=18), "4-byte aligned"),
    (dict(al=18), "4-byte aligned"), (dict(B=65536), "too many sequences")])
def test_accept_refusals(kw, needle):
    rc, msg = _accept(**kw)
    assert rc == -3 and needle in msg and msg.startswith("Paged cache accept failed: "), msg


def test_nothing_to_do_is_not_an_error():
    assert _append(T=0)[0] == 0 and _attend(T=0)[0] == 0 and _accept(A=0)[0] == 0


def test_argument_structs_match_the_header(tmp_path):
    """Sizes and the offsets of each struct's last named field, as a C compiler lays them out."""
    src = tmp_path / "layout.c"
    src.write_text('''#include <stddef.h>
#include <stdio.h>
#include "rdnattention.h"
int main(void) {
    printf("%zu %zu %zu %zu\\n", sizeof(rdna_paged_cache), sizeof(rdna_paged_append_args),
           sizeof(rdna_paged_attention_args), sizeof(rdna_paged_accept_args));
    printf("%zu %zu %zu %zu\\n", offsetof(rdna_paged_cache, dtype), offsetof(rdna_paged_append_args, rope_rows),
           offsetof(rdna_paged_attention_args, scale), offsetof(rdna_paged_accept_args, max_accepted));
    return 0;
}''')
    exe = tmp_path / "layout"
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", f"-I{include}", str(src), "-o", str(exe)], check=True)
    sizes, offsets = ([int(x) for x in line.split()] for line in subprocess.check_output([str(exe)], text=True).splitlines())
    cache = struct.Struct("=" + paged._CACHE)
    assert sizes == [cache.size, paged._APPEND.size, paged._ATTENTION.size, paged._ACCEPT.size]
    assert offsets == [cache.size - 8, paged._APPEND.size - 4, paged._ATTENTION.size - 8, paged._ACCEPT.size - 8]


def test_null_arguments():
    lib = R._lib_handle()
    for call in (lib.rdna_paged_kv_append, lib.rdna_attention_forward_paged, lib.rdna_paged_kv_accept):
        assert call(None, None) == -3
        assert "null arguments" in lib.rdna_get_error().decode()


def test_workspace_size():
    ws = R._lib_handle().rdna_attention_paged_workspace_size
    assert ws(1, 32, 8, 1, 128, 64, 64) % 256 == 0 and ws(1, 32, 8, 1, 128, 64, 64) > 0
    assert ws(1, 32, 8, 16, 128, 64, 64) >= ws(1, 32, 8, 1, 128, 64, 64)
    assert ws(1, 32, 0, 1, 128, 64, 64) == 0 and ws(1, 32, 5, 1, 128, 64, 64) == 0


@pytest.mark.parametrize("call", [_append, _attend])
def test_tables_without_rows_are_refused(call):
    """No position lies inside them, and the kernels' reads start at row 0."""
    rc, msg = call(cos=16, sin=32, rows=0)
    assert rc == -3 and "no rows" in msg, msg


@pytest.mark.parametrize("kw", [dict(B=1 << 15, Hkv=1 << 15, T=1 << 30), dict(B=1 << 15, Hkv=1 << 15, T=1 << 29, D=256)])
def test_append_products_do_not_wrap(kw):
    """2^15 x 2^15 x 2^30 x 128 / 8 chunks are 0 modulo 2^64."""
    rc, msg = _append(**kw)
    assert rc == -3 and "too large for one launch" in msg, msg


@pytest.mark.parametrize("H,T", [(1 << 20, 1 << 19), (1 << 31, 1 << 31), ((1 << 32) - 1, (1 << 32) - 1), (1 << 28, 2)])
def test_attention_products_do_not_wrap(H, T):
    """2^20 heads x 2^19 tokens are 2^32 row tiles, 0 in 32 bits (and once a division by it)."""
    assert R._lib_handle().rdna_attention_paged_workspace_size(1, H, 1, T, 128, 64, 64) == 0
    rc, msg = _attend(B=1, H=H, Hkv=1, T=T)
    assert rc == -3 and "sequence too long" in msg, msg


def test_python_entries_check_their_tensors():
    c = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    t, n = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    with pytest.raises(TypeError):
        R.flash_attn_paged(q, c.numpy(), c, t, n)
    for call in (lambda: R.flash_attn_paged(q, c, c, t, n), lambda: R.paged_kv_append(q, q, c, c, t, n),
                 lambda: R.paged_kv_accept(c, c, t, n, t)):
        with pytest.raises(ValueError, match="CUDA device"):
            call()
    assert R.SUPPORTED_HEAD_DIMS_PAGED == (32, 64, 96, 128, 160, 192, 224, 256)


def test_oracle_against_a_dense_causal_computation():
    g = torch.Generator().manual_seed(0)
    S, T, Hkv, H, D, P = 40, 6, 2, 4, 32, 16
    k, v = (torch.randn(Hkv, S, D, generator=g).half() for _ in range(2))
    q = torch.randn(1, H, T, D, generator=g).half()
    kc, vc = torch.zeros(5, Hkv, P, D).half(), torch.zeros(5, Hkv, P, D).half()
    table = torch.tensor([[3, 0, 4]], dtype=torch.int32)
    kc, _, vc = O.append(k[None], v[None], kc, vc, table, [0])
    got, _ = O.attention(q, kc.half(), vc, table, [S - T])
    kk, vv = k.double().repeat_interleave(2, 0), v.double().repeat_interleave(2, 0)
    s = q[0].double() @ kk.transpose(1, 2) * D ** -0.5
    s = s.masked_fill(torch.arange(S)[None] > torch.arange(S - T, S)[:, None], float("-inf"))
    assert (got[0] - torch.softmax(s, -1) @ vv).abs().max() < 1e-12
    mask = torch.tril(torch.ones(1, T, T, dtype=torch.bool))
    for w in (-1, 1, 3, 20):
        a = O.attention(q, kc.half(), vc, table, [S - T], window=w)[0]
        b = O.attention(q, kc.half(), vc, table, [S - T], mask=mask, window=w)[0]
        assert torch.equal(a, b)
