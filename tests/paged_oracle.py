"""Paged KV-cache operators in 64 bits, written from their definitions, and the
error bounds their kernels are held to.

Attention of row (head, t) of sequence b: o = sum_j p_j v_j / sum_j p_j over the
slots it sees, p_j = exp(scale * q . k_j), q turned to its position.  The bound
for each output element counts the roundings the kernels make, u = eps / 2 of the
cache's type:
  * q is rounded after the turn: the scores move by at most
    d = u * scale * max_j sum_i |q_i k_ji|, plus fp32 products and sums,
    (head_dim + 8) * 2^-23 of the same sum; o moves by expm1(2 d) * A with
    A = sum_j p_j |v_j| / sum_j p_j;
  * p is rounded before the second product: u * A, and where fp16 is subnormal
    2^-25 * sum_j |v_j| / l, l = sum_j exp(s_j - max s) >= 1;
  * fp32 sums over n keys in any order of at most n / 8 + 64 steps, and the
    exponential's error: (n / 8 + 64) * 2^-23 * A;
  * the output's rounding: u * |o| (2^-25 where fp16 is subnormal).
"""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def rotate(x, pos, cos, sin):
    """x [..., n, D] in 64 bits, turned to positions pos [n] by interleaved pairs."""
    c, s = cos.double()[pos], sin.double()[pos]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def tables(rows, D, theta=500000.0):
    ang = torch.arange(rows).double()[:, None] * theta ** (-torch.arange(0, D, 2).double() / D)
    return ang.cos().float(), ang.sin().float()


def slot_rows(cache, table_row, n, num_pages):
    """Slots 0 .. n - 1 of a sequence, [Hkv, n, D] in 64 bits; pages outside the cache read as zeros."""
    P = cache.shape[2]
    out = torch.zeros(cache.shape[1], n, cache.shape[3], dtype=torch.float64)
    for lp in range(-(-n // P)):
        page = int(table_row[lp])
        m = min(P, n - lp * P)
        if 0 <= page < num_pages:
            out[:, lp * P:lp * P + m] = cache[page, :, :m].double()
    return out


def visible(T, L, n, mask, window, hi):
    """bool [T, hi]: slots each token sees."""
    see = torch.zeros(T, hi, dtype=torch.bool)
    for t in range(n):
        new = [u for u in range(n) if (u <= t if mask is None else bool(mask[t, u]))]
        if window > 0:
            ctx = range(max(0, L - max(0, window - len(new))), L)
            new = new[max(0, len(new) - window):]
        else:
            ctx = range(L)
        for j in ctx:
            if j < hi:
                see[t, j] = True
        for u in new:
            if L + u < hi:
                see[t, L + u] = True
    return see


def attention(q, k_cache, v_cache, table, lens, news=None, mask=None, positions=None, cos=None, sin=None, window=-1,
              scale=None):
    """(o, bound), both float64 [B, H, T, D]; CPU tensors; mask [B, T, T] or None."""
    B, H, T, D = q.shape
    num_pages, Hkv, P, _ = k_cache.shape
    cap = table.shape[1] * P
    G = H // Hkv
    u, tiny = U[q.dtype], TINY[q.dtype]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, H, T, D, dtype=torch.float64)
    bound = torch.full((B, H, T, D), 1e-30, dtype=torch.float64)
    for b in range(B):
        L = min(max(int(lens[b]), 0), cap)
        n = T if news is None else min(max(int(news[b]), 0), T)
        hi = min(L + n, cap)
        if n == 0 or hi == 0:
            continue
        k, v = slot_rows(k_cache, table[b], hi, num_pages), slot_rows(v_cache, table[b], hi, num_pages)
        see = visible(T, L, n, None if mask is None else mask[b], window, hi)
        pos = torch.tensor([L + t for t in range(T)]) if positions is None else positions[b].long()
        good = torch.ones(T, dtype=torch.bool)
        x = q[b].double()
        if cos is not None:
            good = (pos >= 0) & (pos < cos.shape[0])
            x = rotate(x, pos.clamp(0, cos.shape[0] - 1), cos, sin)
        see &= good[:, None]
        see[n:] = False
        kk, vv = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
        s = scale * x @ kk.transpose(1, 2)
        mag = abs(scale) * x.abs() @ kk.abs().transpose(1, 2)
        s = s.masked_fill(~see, float("-inf"))
        m = s.amax(-1, keepdim=True)
        some = torch.isfinite(m)
        p = torch.where(see, (s - torch.where(some, m, 0.0)).exp(), 0.0)
        l = p.sum(-1, keepdim=True).clamp(min=1e-300)
        o, A = p @ vv / l, p @ vv.abs() / l
        keys = see.sum(-1)[None, :, None].double()
        worst = torch.where(see, mag, 0.0).amax(-1, keepdim=True)
        d = worst * ((u if cos is not None else 0.0) + (D + 8) * 2.0 ** -23)
        seen_v = see.double() @ vv.abs()
        tol = (u * o.abs() + tiny + (u + torch.expm1(2 * d) + (keys / 8 + 64) * 2.0 ** -23) * A
               + tiny * seen_v / l)
        out[b] = torch.where(some, o, 0.0)
        bound[b] = torch.where(some, tol, bound[b])
    return out, bound


def append(key, value, k_cache, v_cache, table, lens, news=None, positions=None, cos=None, sin=None):
    """(K, bound of K, V): the caches after the call, K and its bound in 64 bits, V bit for bit."""
    B, Hkv, T, D = key.shape
    num_pages, _, P, _ = k_cache.shape
    cap = table.shape[1] * P
    K, V = k_cache.double(), v_cache.clone()
    bound = torch.zeros_like(K)
    u, tiny = U[key.dtype], TINY[key.dtype]
    for b in range(B):
        L = min(max(int(lens[b]), 0), cap)
        n = T if news is None else min(max(int(news[b]), 0), T)
        for t in range(n):
            slot = L + t
            if slot >= cap:
                continue
            page, row = int(table[b, slot // P]), slot % P
            pos = L + t if positions is None else int(positions[b, t])
            if not 0 <= page < num_pages or cos is not None and not 0 <= pos < cos.shape[0]:
                continue
            x = key[b, :, t].double()
            V[page, :, row] = value[b, :, t]
            if cos is None:
                K[page, :, row] = x
                continue
            c, s = cos[pos].double(), sin[pos].double()
            a, d = x[:, 0::2], x[:, 1::2]
            y = torch.stack((a * c - d * s, a * s + d * c), -1).flatten(-2)
            mag = torch.stack(((a * c).abs() + (d * s).abs(), (a * s).abs() + (d * c).abs()), -1).flatten(-2)
            K[page, :, row] = y
            bound[page, :, row] = u * y.abs() + tiny + 2.0 ** -22 * mag
    return K, bound, V


def accept(k_cache, v_cache, table, lens, accepted, accepted_lens=None):
    """The caches after the call."""
    num_pages, _, P, _ = k_cache.shape
    cap = table.shape[1] * P
    K, V = k_cache.clone(), v_cache.clone()

    def place(b, slot):
        if not 0 <= slot < cap:
            return None
        page = int(table[b, slot // P])
        return (page, slot % P) if 0 <= page < num_pages else None

    for b in range(table.shape[0]):
        L = min(max(int(lens[b]), 0), cap)
        n = accepted.shape[1] if accepted_lens is None else min(max(int(accepted_lens[b]), 0), accepted.shape[1])
        for i in range(n):
            a = int(accepted[b, i])
            src, dst = place(b, L + a) if a >= 0 else None, place(b, L + i)
            if src is not None and dst is not None:
                K[dst[0], :, dst[1]] = k_cache[src[0], :, src[1]]
                V[dst[0], :, dst[1]] = v_cache[src[0], :, src[1]]
    return K, V
