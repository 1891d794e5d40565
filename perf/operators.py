"""Workloads of the paged KV-cache operators: append, attention, accept.

A serving step with drafted tokens is three calls on one paged cache:
``paged_kv_append`` writes the new tokens' keys (rotated on the way) and
values, ``flash_attn_paged`` lets the new tokens attend to the cache and to
their ancestors in the draft tree, ``paged_kv_accept`` moves the accepted
path to the front.  Each case is one pass through one of them.

``run`` computes an operator in its plain form (elementary torch operations in
32 bits, rounded once at the end), or, with ``own`` set, through the
framework's entry points.
"""
import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of one sequence: the smallest launch, where latency counts
        dict(name="append step b1", op="append", dtype="fp16", B=1, Hkv=8, D=128, T=1, ctx=4096, page=64,
             ragged=False, rope=True, tree=False),
        # the drafted trees of a padded batch, each sequence with its own number of tokens
        dict(name="append tree ragged", op="append", dtype="bf16", B=16, Hkv=3, D=96, T=61, ctx=777, page=16,
             ragged=True, rope=True, tree=True),
        # prompts entering the cache
        dict(name="append prompt", op="append", dtype="fp16", B=4, Hkv=8, D=128, T=4096, ctx=512, page=64,
             ragged=False, rope=True, tree=False),
        # one token of one sequence over a short context: latency
        dict(name="attend step b1", op="attend", dtype="fp16", B=1, H=32, Hkv=8, D=128, T=1, ctx=4096, page=64,
             ragged=False, rope=True, tree=False, window=-1),
        # the decode workload over long contexts, now through page tables
        dict(name="attend step b64", op="attend", dtype="fp16", B=64, H=64, Hkv=8, D=128, T=1, ctx=32768, page=64,
             ragged=False, rope=False, tree=False, window=-1),
        # ordinary ragged decode batch, small pages
        dict(name="attend step ragged", op="attend", dtype="bf16", B=33, H=32, Hkv=8, D=128, T=1, ctx=8192, page=16,
             ragged=True, rope=True, tree=False, window=-1),
        # one sequence verifying a small tree
        dict(name="attend tree b1", op="attend", dtype="bf16", B=1, H=32, Hkv=8, D=128, T=16, ctx=8192, page=16,
             ragged=False, rope=True, tree=True, window=-1),
        # a batch verifying large trees (256 query rows to each key and value head)
        dict(name="attend tree b16", op="attend", dtype="fp16", B=16, H=32, Hkv=8, D=128, T=64, ctx=8192, page=64,
             ragged=True, rope=True, tree=True, window=-1),
        # odd everything: head count, width, tree, an empty context, a sliding window
        dict(name="attend tree odd", op="attend", dtype="bf16", B=5, H=15, Hkv=3, D=96, T=13, ctx=5001, page=16,
             ragged=True, rope=True, tree=True, window=1000),
        # a chunk of a long prompt over what the cache holds already: compute-bound
        dict(name="attend chunk", op="attend", dtype="fp16", B=2, H=32, Hkv=8, D=128, T=512, ctx=16384, page=128,
             ragged=False, rope=True, tree=False, window=-1),
        # the accepted path of one sequence
        dict(name="accept b1", op="accept", dtype="fp16", B=1, Hkv=8, D=128, T=16, A=4, ctx=1024, page=64,
             ragged=False),
        # a batch of sequences, each accepting its own number of tokens
        dict(name="accept b64", op="accept", dtype="bf16", B=64, Hkv=8, D=128, T=64, A=9, ctx=1000, page=16,
             ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "accept"])
    case = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), B=_log(rng, 1, 64), Hkv=rng.choice([1, 2, 3, 4, 5, 8]),
                D=rng.choice([32, 64, 96, 128, 128, 128, 160, 192, 256]),
                page=rng.choice([8, 16, 16, 32, 64, 64, 72, 100, 128, 256]), ragged=rng.random() < 0.6)
    if op == "append":
        case.update(T=_log(rng, 1, 4096), ctx=_log(rng, 1, 4096), rope=rng.random() < 0.8, tree=False)
        case["tree"] = case["T"] <= 256 and rng.random() < 0.5
        while case["B"] * case["Hkv"] * case["D"] * (case["T"] + case["ctx"]) > 18_000_000 and case["B"] > 1:
            case["B"] = max(1, case["B"] // 2)
    elif op == "attend":
        tree = rng.random() < 0.6
        case.update(H=case["Hkv"] * rng.choice([1, 2, 3, 4, 5, 8]), T=_log(rng, 1, 128 if tree else 512),
                    ctx=_log(rng, 1, 32768), rope=rng.random() < 0.7, tree=tree,
                    window=rng.choice([-1, -1, -1, 256, 1000, 4096]))
        while case["B"] > 1 and (case["B"] * case["Hkv"] * case["D"] * case["ctx"] > 400_000_000
                                 or case["B"] * case["H"] * case["T"] * case["D"] * case["ctx"] > 30_000_000_000):
            case["B"] = max(1, case["B"] // 2)
    else:
        case.update(T=_log(rng, 2, 128), ctx=_log(rng, 1, 2048))
        case["A"] = rng.randint(1, min(16, case["T"]))
    return case


# ------------------------------------------------------------- the lengths
def _lens(case):
    """Tokens in the cache before the call, for each sequence (a ragged batch holds an empty one)."""
    B, ctx = case["B"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * B
    return [ctx * ((b * 6 + 16) % 17) // 16 for b in range(B)]


def _news(case):
    """New tokens of each sequence, at most T (the batch is padded to T)."""
    B, T = case["B"], case["T"]
    if not case["ragged"]:
        return [T] * B
    return [T - (b * 5 % 8) * T // 8 for b in range(B)]


def _accepts(case):
    """Accepted tokens of each sequence, at most A."""
    if not case["ragged"]:
        return [case["A"]] * case["B"]
    return [min(case["A"] - b % 4 * case["A"] // 4, n) for b, n in enumerate(_news(case))]


def _spans(case):
    """Keys of the old context that some new token of each sequence sees."""
    w = case.get("window", -1)
    return [n if w <= 0 else min(n, w - 1) for n in _lens(case)]


# -------------------------------------------------------------- the inputs
def _tree(case, seed):
    """Random draft trees: (mask bool [B, T, T], depth [B, T]); token t sees itself and its ancestors."""
    B, T = case["B"], case["T"]
    g = torch.Generator().manual_seed(seed + 101)
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    depth = torch.zeros(B, T, dtype=torch.int64)
    for t in range(T):
        if t > 0:
            # a parent among the last few tokens of the level order
            lo = max(0, t - 1 - max(4, t // 2))
            par = torch.randint(lo, t, (B,), generator=g)
            rows = torch.arange(B)
            mask[:, t] = mask[rows, par]
            depth[:, t] = depth[rows, par] + 1
        mask[:, t, t] = True
    return mask, depth


def _pages(case, seed):
    """(page table [B, max_pages], number of pages): the sequences' pages in random order, a few spare ones between."""
    P = case["page"]
    need = [max(1, -(-(n + case["T"]) // P)) for n in _lens(case)]
    g = torch.Generator().manual_seed(seed + 202)
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, dtype=torch.int64).to(torch.int32)
    table = torch.zeros(case["B"], max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    dev = torch.device("cuda")
    dt = _DTYPES[case["dtype"]]
    B, Hkv, D, T, P = case["B"], case["Hkv"], case["D"], case["T"], case["page"]
    lens, news = _lens(case), _news(case)
    g = torch.Generator(device=dev).manual_seed(seed)
    table, total = _pages(case, seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    st = {"case": case, "lens": lens, "news": news, "k_cache": randn(total, Hkv, P, D),
          "v_cache": randn(total, Hkv, P, D), "page_table": table.to(dev),
          "cache_lens": torch.tensor(lens, dtype=torch.int32, device=dev),
          "new_lens": torch.tensor(news, dtype=torch.int32, device=dev) if case["ragged"] else None}
    if case["op"] == "accept":
        gc = torch.Generator().manual_seed(seed + 303)
        accepts = _accepts(case)
        path = torch.zeros(B, case["A"], dtype=torch.int32)
        for b, n in enumerate(accepts):
            # the path starts at the first drafted token and then runs through tokens behind the
            # accepted ones, so that a second pass finds the same sources
            far = torch.randperm(max(news[b] - n, 0), generator=gc)[:max(n - 1, 0)].sort().values + n
            for i in range(n):
                path[b, i] = int(far[i - 1]) if 0 < i <= far.numel() else i
        st.update(accepts=accepts, path=path, accepted=path.to(dev),
                  accepted_lens=torch.tensor(accepts, dtype=torch.int32, device=dev))
        return st
    depth = None
    st["tree_mask"] = None
    if case["tree"]:
        mask, depth = _tree(case, seed)
        st["tree_mask"] = mask.to(dev)
    st["positions"] = None
    if depth is not None:
        st["positions"] = (torch.tensor(lens)[:, None] + depth).to(torch.int32).to(dev)
    st["cos"] = st["sin"] = None
    if case["rope"]:
        pos = torch.arange(case["ctx"] + T, dtype=torch.float64, device=dev)[:, None]
        ang = pos * 500000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
        st["cos"], st["sin"] = ang.cos().float().contiguous(), ang.sin().float().contiguous()
    if case["op"] == "append":
        st["key"], st["value"] = randn(B, Hkv, T, D), randn(B, Hkv, T, D)
    else:
        st["query"] = randn(B, case["H"], T, D) * 2  # peaked rows, as trained heads have them
    return st


# ------------------------------------------------------------ the plain forms
def _positions(st, b):
    if st["positions"] is not None:
        return st["positions"][b].long()
    return st["lens"][b] + torch.arange(st["case"]["T"], device="cuda")


def _rotate(x, cos, sin):
    """Interleaved pairs of the last axis of x [heads, tokens, D]; cos/sin [tokens, D/2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)


def _slots(st, b, first, count):
    """(pages, rows) of the slots first .. first + count - 1 of sequence b."""
    s = torch.arange(first, first + count, device="cuda")
    P = st["case"]["page"]
    return st["page_table"][b].long()[s // P], s % P


def _plain_append(st):
    kc, vc = st["k_cache"], st["v_cache"]
    for b, n in enumerate(st["news"]):
        if n == 0:
            continue
        k, v = st["key"][b, :, :n].float(), st["value"][b, :, :n]
        if st["cos"] is not None:
            pos = _positions(st, b)[:n]
            k = _rotate(k, st["cos"][pos], st["sin"][pos])
        pages, rows = _slots(st, b, st["lens"][b], n)
        kc[pages, :, rows] = k.to(kc.dtype).transpose(0, 1)
        vc[pages, :, rows] = v.transpose(0, 1)
    return kc, vc


def _visible(st, b):
    """bool [n, len + n]: what the n new tokens of sequence b see."""
    case, L, n = st["case"], st["lens"][b], st["news"][b]
    w = case["window"]
    qpos = _positions(st, b)[:n]
    kpos = torch.cat((torch.arange(L, device="cuda"), qpos))
    if st["tree_mask"] is not None:
        new = st["tree_mask"][b, :n, :n]
    else:
        new = torch.arange(n, device="cuda")[:, None] >= torch.arange(n, device="cuda")[None, :]
    seen = torch.cat((torch.ones(n, L, dtype=torch.bool, device="cuda"), new), dim=1)
    if w > 0:
        seen = seen & (qpos[:, None] - kpos[None, :] < w)
    return seen


def _plain_attend(st):
    case, q = st["case"], st["query"]
    out = torch.zeros_like(q)
    G = case["H"] // case["Hkv"]
    for b, n in enumerate(st["news"]):
        if n == 0:
            continue
        L = st["lens"][b]
        qb = q[b, :, :n].float()
        if st["cos"] is not None:
            pos = _positions(st, b)[:n]
            qb = _rotate(qb, st["cos"][pos], st["sin"][pos])
        pages, rows = _slots(st, b, 0, L + n)
        k = st["k_cache"][pages, :, rows].transpose(0, 1).float()
        v = st["v_cache"][pages, :, rows].transpose(0, 1).float()
        qb = qb.reshape(case["Hkv"], G * n, case["D"])
        s = (qb @ k.transpose(1, 2)) * case["D"] ** -0.5
        seen = _visible(st, b).repeat(G, 1)
        s = s.masked_fill(~seen, float("-inf"))
        m = s.amax(dim=-1, keepdim=True)
        p = (s - m).exp()
        o = (p @ v) / p.sum(dim=-1, keepdim=True)
        out[b, :, :n] = o.reshape(case["H"], n, case["D"]).to(out.dtype)
    return out


def _plain_accept(st):
    kc, vc = st["k_cache"], st["v_cache"]
    for b, n in enumerate(st["accepts"]):
        if n == 0:
            continue
        L, P = st["lens"][b], st["case"]["page"]
        src = L + st["accepted"][b, :n].long()
        sp, sr = st["page_table"][b].long()[src // P], src % P
        dp, dr = _slots(st, b, L, n)
        kc[dp, :, dr] = kc[sp, :, sr]
        vc[dp, :, dr] = vc[sp, :, sr]
    return kc, vc


def run(state):
    op = state["case"]["op"]
    if own:
        import rdnattention_b200 as R

        if op == "append":
            return R.paged_kv_append(state["key"], state["value"], state["k_cache"], state["v_cache"],
                                     state["page_table"], state["cache_lens"], new_lens=state["new_lens"],
                                     positions=state["positions"], rot_cos=state["cos"], rot_sin=state["sin"])
        if op == "attend":
            return R.flash_attn_paged(state["query"], state["k_cache"], state["v_cache"], state["page_table"],
                                      state["cache_lens"], new_lens=state["new_lens"], tree_mask=state["tree_mask"],
                                      positions=state["positions"], rot_cos=state["cos"], rot_sin=state["sin"],
                                      window_size=state["case"]["window"])
        return R.paged_kv_accept(state["k_cache"], state["v_cache"], state["page_table"], state["cache_lens"],
                                 state["accepted"], accepted_lens=state["accepted_lens"])
    return {"append": _plain_append, "attend": _plain_attend, "accept": _plain_accept}[op](state)


# ------------------------------------------------------------------ the work
def work(case):
    esz = 2
    B, Hkv, D, T = case["B"], case["Hkv"], case["D"], case["T"]
    row = Hkv * D * esz  # one token's keys (or values)
    if case["op"] == "append":
        n = sum(_news(case))
        tables = (n * D * 4 if case["rope"] else 0) + (n * 4 if case["tree"] else 0)
        return {"bytes": 4 * n * row + tables + 8 * B, "flops": 3 * n * Hkv * D if case["rope"] else 0}
    if case["op"] == "accept":
        n = sum(_accepts(case))
        return {"bytes": 4 * n * row + 4 * n + 8 * B, "flops": 0}
    news, spans = _news(case), _spans(case)
    keys = sum(s + n for s, n in zip(spans, news) if n > 0)
    # the old context for every row; of the new tokens a chain sees the triangle, a tree at least itself
    pairs = sum(n * s + (n if case["tree"] else n * (n + 1) // 2) for s, n in zip(spans, news))
    io = 2 * sum(news) * case["H"] * D * esz
    mask = sum(n * n for n in news) if case["tree"] else 0
    return {"bytes": 2 * keys * row + io + mask, "flops": 4 * pairs * case["H"] * D}


# -------------------------------------------------- the definition in 64 bits
def _turn(x, pos, cos, sin):
    """One token [heads, D] turned to its position: each pair as a complex number times cos + i sin."""
    z = torch.view_as_complex(x.double().reshape(x.shape[0], -1, 2).contiguous())
    turned = z * torch.complex(cos[pos].double(), sin[pos].double())
    return torch.view_as_real(turned).reshape(x.shape)


def exact(case, seed):
    if case["op"] == "attend":
        pairs = sum(n * (s + n) for s, n in zip(_lens(case), _news(case))) * case["H"] * case["D"]
        if pairs > 1.5e11:
            return None
    st = prepare(case, seed)
    P, table = case["page"], st["page_table"].tolist()
    if case["op"] == "accept":
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        old_k, old_v = kc.clone(), vc.clone()
        for b, n in enumerate(st["accepts"]):
            for i in range(n):
                to, fr = st["lens"][b] + i, st["lens"][b] + int(st["path"][b, i])
                kc[table[b][to // P], :, to % P] = old_k[table[b][fr // P], :, fr % P]
                vc[table[b][to // P], :, to % P] = old_v[table[b][fr // P], :, fr % P]
        return kc, vc
    if case["op"] == "append":
        if sum(st["news"]) > 20000:
            return None
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        for b, n in enumerate(st["news"]):
            if n == 0:
                continue
            slot = torch.arange(st["lens"][b], st["lens"][b] + n)
            page = torch.tensor(table[b])[slot // P].to(kc.device)
            line = (slot % P).to(kc.device)
            k = st["key"][b, :, :n].double()
            if case["rope"]:
                pos = slot.to(kc.device) if st["positions"] is None else st["positions"][b, :n].long()
                z = torch.view_as_complex(k.reshape(case["Hkv"], n, -1, 2).contiguous())
                turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())
                k = torch.view_as_real(z * turn).reshape(case["Hkv"], n, case["D"])
            kc[page, :, line] = k.transpose(0, 1)
            vc[page, :, line] = st["value"][b, :, :n].double().transpose(0, 1)
        return kc, vc
    H, Hkv, D, T, w = case["H"], case["Hkv"], case["D"], case["T"], case["window"]
    out = torch.zeros(case["B"], H, T, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["news"]):
        L = st["lens"][b]
        if n == 0:
            continue
        slot = torch.arange(L + n, device="cuda")
        page = st["page_table"][b].long()[slot // P]
        k = st["k_cache"][page, :, slot % P].double()  # [L + n, Hkv, D]
        v = st["v_cache"][page, :, slot % P].double()
        for t0 in range(0, n, 128):
            ts = range(t0, min(n, t0 + 128))
            rows, seen = [], []
            for t in ts:
                pos = L + t if st["positions"] is None else int(st["positions"][b, t])
                x = st["query"][b, :, t].double()
                rows.append(_turn(x, pos, st["cos"], st["sin"]) if case["rope"] else x)
                see = torch.ones(L + n, dtype=torch.bool, device="cuda")
                see[L:] = st["tree_mask"][b, t, :n] if case["tree"] else torch.arange(n, device="cuda") <= t
                if w > 0:
                    at = slot.clone()
                    if st["positions"] is not None:
                        at[L:] = st["positions"][b, :n]
                    see &= pos - at < w
                seen.append(see)
            x = torch.stack(rows, dim=1).reshape(Hkv, H // Hkv, len(rows), D)  # heads, tokens
            logit = torch.einsum("hgtd,jhd->hgtj", x, k) / math.sqrt(D)
            logit = torch.where(torch.stack(seen), logit, torch.full_like(logit, -math.inf))
            prob = torch.softmax(logit, dim=-1)
            out[b, :, ts.start:ts.stop] = torch.einsum("hgtj,jhd->hgtd", prob, v).reshape(H, len(rows), D)
    return out
