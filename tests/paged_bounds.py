"""The paged attention in 64 bits with a bound that counts what the kernels keep of the query
after the turn, inputs on which single keys, bits and rescales count, and the schedule of the
kernels' work (for choosing sizes).

The bound of an output element, u = eps / 2 of the cache's type, t = 2^-25 where it is fp16
(half its smallest step) and 0 else:
  * the turn in 32 bits: 2^-23 (|x c| + |y s|) for each component a of the query;
  * a as hi + lo, both of the cache's type: hi leaves at most u |a| (where |a| passes fp16's
    largest value, |a| - 65504), lo is off by u of what hi left, or t;
  * a score is a sum of 2 D products (D without tables), exact in 32 bits, in any order, each
    step off by at most 2^-23 of sum_i |a_i k_i|; its scaling and the subtraction of the
    reference 4 steps more.  With d the largest of all this over the row's visible keys,
    times |scale|, the weights are off by a factor of at most exp(2 d);
  * p is rounded before the second product: u of it, or t against a reference that is at most
    the largest score M_j of the slots up to j's tile's end, j + 63 at most: t exp(M_j - max s);
  * 32-bit sums over n keys in any order of at most n / 8 + 64 steps, and the exponential's
    error: (n / 8 + 64) 2^-23;
  * the output's rounding: u |o| or t.
With A = sum_j p_j |v_j| / l and l = sum_j p_j, p_j = exp(s_j - max s):
  u |o| + t + (u + expm1(2 d) + (n / 8 + 64) 2^-23) A + t sum_j exp(M_j - max s) |v_j| / l.
"""
import torch

import paged_oracle as O

F16, BF16 = torch.float16, torch.bfloat16
MAX = {F16: 65504.0, BF16: torch.finfo(BF16).max}


def attention(q, k_cache, v_cache, table, lens, news=None, mask=None, positions=None, cos=None, sin=None, window=-1,
              scale=None, plant=None, hide=None):
    """(o, bound), float64 [B, H, T, D]; arguments as paged_oracle.attention.  plant="lo": the mistake of
    rounding the turned query once; hide=(b, slot): the mistake of not seeing that slot."""
    B, H, T, D = q.shape
    num_pages, Hkv, P, _ = k_cache.shape
    cap, G = table.shape[1] * P, H // Hkv
    u, t = O.U[q.dtype], O.TINY[q.dtype]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, H, T, D, dtype=torch.float64)
    bound = torch.full((B, H, T, D), 1e-30, dtype=torch.float64)
    for b in range(B):
        L = min(max(int(lens[b]), 0), cap)
        n = T if news is None else min(max(int(news[b]), 0), T)
        hi = min(L + n, cap)
        if n == 0 or hi == 0:
            continue
        k, v = O.slot_rows(k_cache, table[b], hi, num_pages), O.slot_rows(v_cache, table[b], hi, num_pages)
        see = O.visible(T, L, n, None if mask is None else mask[b], window, hi)
        if hide is not None and hide[0] == b:
            see[:, hide[1]] = False
        pos = torch.arange(L, L + T) if positions is None else positions[b].long()
        x = q[b].double()
        turned = torch.zeros_like(x)
        if cos is not None:
            good = (pos >= 0) & (pos < cos.shape[0])
            see &= good[:, None]
            at = pos.clamp(0, cos.shape[0] - 1)
            c, s = cos.double()[at].repeat_interleave(2, -1), sin.double()[at].repeat_interleave(2, -1)
            other = x.reshape(*x.shape[:-1], -1, 2).flip(-1).flatten(-2)
            turned = 2.0 ** -23 * ((x * c).abs() + (other * s).abs())
            x = O.rotate(x, at, cos, sin)
            left = torch.maximum(u * x.abs(), x.abs() - MAX[q.dtype])
            turned += torch.clamp(u * left, min=t)
            if plant == "lo":
                x = x.to(q.dtype).double()
        see[n:] = False
        kk, vv = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
        sc = scale * x @ kk.transpose(1, 2)
        steps = (D if cos is None else 2 * D) + 4
        d = abs(scale) * (turned + steps * 2.0 ** -23 * x.abs()) @ kk.abs().transpose(1, 2)
        d = torch.where(see, d, 0.0).amax(-1, keepdim=True)
        sc = sc.masked_fill(~see, float("-inf"))
        m = sc.amax(-1, keepdim=True)
        some = torch.isfinite(m)
        p = torch.where(see, (sc - torch.where(some, m, 0.0)).exp(), 0.0)
        l = p.sum(-1, keepdim=True).clamp(min=1e-300)
        # M_j: the running maximum, 63 slots on
        late = torch.nn.functional.pad(sc, (0, 63), value=float("-inf")).cummax(-1).values[..., 63:]
        late = (late - torch.where(some, m, 0.0)).exp()
        o, A = p @ vv / l, p @ vv.abs() / l
        keys = see.sum(-1)[None, :, None].double()
        tol = (u * o.abs() + t + (u + torch.expm1(2 * d) + (keys / 8 + 64) * 2.0 ** -23) * A
               + t * (torch.where(see, late, 0.0) @ vv.abs()) / l)
        out[b] = torch.where(some, o, 0.0)
        bound[b] = torch.where(some, tol, bound[b])
    return out, bound


# ------------------------------------------------------------------- inputs
def pages_for(g, lens, T, P, spare=2):
    """(table, pages): room for T more tokens each, pages in random order."""
    need = [max(1, -(-(n + T) // P)) for n in lens]
    perm = torch.randperm(sum(need) + spare, generator=g).int()
    table, at = torch.full((len(lens), max(need)), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, sum(need) + spare


def put(cache, table, b, slot, h, row):
    P = cache.shape[2]
    cache[table[b, slot // P], h, slot % P] = row


def split_case(dtype, D, T, P, mag=400.0):
    """Each token sees two keys of its own among the drafted slots, both orthogonal to its turned
    query and along the signs of what its rounding leaves, one for it and one against: without lo the
    scores move apart by about u / 2 of sum |a k| = mag, with it they stay equal.  T even; the second
    half of the tokens see nothing.  Values +1 and -1."""
    g = torch.Generator().manual_seed(D + T)
    H = 2
    table, pages = pages_for(g, [0], T, P)
    kc = torch.zeros(pages, H, P, D, dtype=dtype)
    vc = torch.zeros_like(kc)
    q = torch.randn(1, H, T, D, generator=g).to(dtype)
    cos, sin = O.tables(T + 1000, D)
    pos = torch.randint(0, T + 1000, (1, T), generator=g).int()
    mask = torch.zeros(1, T, T, dtype=torch.bool)
    for t in range(T // 2):
        mask[0, t, 2 * t:2 * t + 2] = True
        for h in range(H):
            a = O.rotate(q[0, h, t:t + 1].double(), pos[0, t:t + 1].long(), cos, sin)[0]
            sign = (a - a.to(dtype).double()).sign()
            k = sign - (a @ sign) / (a @ a) * a
            k = (k * mag / (a.abs() @ k.abs()) * D ** 0.5).to(dtype)  # (times D^-1/2, the scale)
            put(kc, table, 0, 2 * t, h, k)
            put(kc, table, 0, 2 * t + 1, h, -k)
            put(vc, table, 0, 2 * t, h, torch.ones(D))
            put(vc, table, 0, 2 * t + 1, h, -torch.ones(D))
    return dict(q=q, k_cache=kc, v_cache=vc, table=table, lens=[0], mask=mask, positions=pos, cos=cos, sin=sin)


def telling_slots(L, n, P, D, lo=0):
    """Up to D slots of [lo, L + n) at which a schedule or a mask can go wrong, by importance."""
    hi, at = L + n, []

    def add(*slots):
        for s in slots:
            if lo <= s < hi and s not in at:
                at.append(s)

    add(lo, lo + 1, L - 1, L, L + 1, hi - 1, hi - 2)
    for s in list(range(P, hi, P))[-3:] + list(range(P, hi, P))[:3]:
        add(s - 1, s)
    tiles = list(range(64, hi, 64))
    for s in tiles[:: max(1, len(tiles) // (D // 4))]:
        add(s - 1, s)
    for s in range(L, hi):
        add(s)
    for s in range(lo, hi, max(1, (hi - lo) // D)):
        add(s)
    return at[:D]


def telling_case(dtype, H, Hkv, T, D, P, lens, kind="chain", window=-1):
    """Scores of zero (keys of zero) and values of zero but for one column each in up to D slots per
    sequence: an output column is value / number of visible keys where its slot is seen, else zero."""
    g = torch.Generator().manual_seed(D + T + P)
    B = len(lens)
    table, pages = pages_for(g, lens, T, P)
    kc = torch.zeros(pages, Hkv, P, D, dtype=dtype)
    vc = torch.zeros_like(kc)
    q = torch.randn(B, H, T, D, generator=g).to(dtype)
    slots = []
    for b, L in enumerate(lens):
        lo = max(0, L - window) if window > 0 else 0
        slots.append(telling_slots(L, T, P, D, lo))
        for i, s in enumerate(slots[-1]):
            row = torch.zeros(D)
            row[i] = 2.0 ** 15
            for h in range(Hkv):
                put(vc, table, b, s, h, row)
    mask = None
    if kind == "tree":
        mask = torch.rand(B, T, T, generator=g) < 0.5
    return dict(q=q, k_cache=kc, v_cache=vc, table=table, lens=lens, mask=mask, window=window), slots


def rising_case(dtype, H, Hkv, T, D, P, lens, pattern, step, rows="all", rope=False):
    """Keys whose scores rise by `step` (in powers of two) from tile to tile of 64: level = tile number
    ("every"), half of it ("second"), 0 but from the context's last tile on ("end"); values shrink alike, so that every
    tile has the same weight in the output.  rows: which rows rise, "all", "odd" heads or tokens below
    half ("warps"); the others' scores do not.  fp16 values hold three levels, 0 to 2."""
    g = torch.Generator().manual_seed(D + T + int(step) + len(pattern))
    B, most = len(lens), 2 if dtype == F16 else 12
    table, pages = pages_for(g, lens, T, P)
    kc = (0.2 * torch.randn(pages, Hkv, P, D, generator=g)).to(dtype)
    vc = torch.zeros(pages, Hkv, P, D, dtype=dtype)
    top = 14 if dtype == F16 else 60
    for b, L in enumerate(lens):
        last = L // 64
        for s in range(L + T):
            tile = s // 64
            level = {"every": tile, "second": tile // 2, "end": int(tile >= last)}[pattern]
            level = min(level, most)
            for h in range(Hkv):
                row = kc[table[b, s // P], h, s % P]
                row[0] = level * step * 0.6931471805599453
                row[1] = 0.0
                put(vc, table, b, s, h, (1 + 0.5 * torch.randn(D, generator=g)) * 2.0 ** (top - step * level))
    q = 0.2 * torch.randn(B, H, T, D, generator=g)
    q[..., 0], q[..., 1] = 1.0, 0.0
    still = torch.zeros(H, T, dtype=torch.bool)
    if rows == "odd":
        still[::2] = True
    elif rows == "warps":
        still[:, :T // 2] = True
    q[..., 0] = torch.where(still, 0.0, q[..., 0])
    case = dict(q=q.to(dtype), k_cache=kc, v_cache=vc, table=table, lens=lens, scale=1.0)
    if rope:  # a turn by nothing, as the tables of position 0 are
        cos, sin = O.tables(1, D)
        case.update(cos=cos, sin=sin, positions=torch.zeros(B, T, dtype=torch.int32))
    return case


def draft_tree(g, B, T):
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


def plain_case(dtype, H, Hkv, T, D, P, lens, kind="chain", window=-1, rope=True, news=None, scale=None):
    """Random queries, keys and values."""
    g = torch.Generator().manual_seed(3 * D + T + P + len(lens))
    B = len(lens)
    table, pages = pages_for(g, lens, T, P)
    case = dict(q=(2 * torch.randn(B, H, T, D, generator=g)).to(dtype),
                k_cache=torch.randn(pages, Hkv, P, D, generator=g).to(dtype),
                v_cache=torch.randn(pages, Hkv, P, D, generator=g).to(dtype), table=table, lens=lens, window=window,
                news=news, scale=scale)
    if kind == "tree":
        case["mask"], depth = draft_tree(g, B, T)
        case["positions"] = (torch.tensor(lens)[:, None] + depth).int()
    if rope:
        case["cos"], case["sin"] = O.tables(max(lens) + T + 1, D)
    return case


# ----------------------------------------------------------------- schedule
def segments(B, H, Hkv, T, D, P, lens, window=-1, kind="chain", ctas=148):
    """The list of a launch cut among its CTAs: for each CTA the (unit, tiles, tiles of the unit) of its
    segments with tiles, in order.  A unit is (row tile, sequence, KV head); D up to 128."""
    rows = H // Hkv * T
    RT, W = (128, 12) if rows > 16 else (16, 6)
    tpp = -(-P // 64) if P >= 64 else 0

    def tile_of(j):
        return j // P * tpp + j % P // 64 if tpp else j // 64

    starts, pos = [], 0
    for rt in range(-(-rows // RT)):
        for b, L in enumerate(lens):
            ta, tb = rt * RT * Hkv // H, min((min((rt + 1) * RT, rows) - 1) * Hkv // H, T - 1)
            hi = L + T if kind == "tree" else L + tb + 1
            lo = max(0, (L if kind == "tree" else L + ta + 1) - window) if window > 0 else 0
            n = tile_of(hi - 1) + 1 - tile_of(lo)
            for h in range(Hkv):
                starts.append(((rt, b, h), pos, n))
                pos += W + n
    ctas = min(ctas, pos)
    q, r = divmod(pos, ctas)
    out = [[] for _ in range(ctas)]
    for unit, at, n in starts:
        for c in range(ctas):
            begin, end = c * q + min(c, r), (c + 1) * q + min(c + 1, r)
            k = min(at + W + n, end) - max(at + W, begin)
            if k > 0:
                out[c].append((unit, k, n))
    return out
