"""Paged KV cache: append with the position rotation, attention for single
tokens, chains and drafted trees, and moving the accepted tokens to the front.

One serving step, the cache lengths untouched until its end:

    >>> paged_kv_append(k, v, k_cache, v_cache, table, lens, positions=pos, rot_cos=cos, rot_sin=sin)
    >>> o = flash_attn_paged(q, k_cache, v_cache, table, lens, tree_mask=mask, positions=pos,
    ...                      rot_cos=cos, rot_sin=sin)
    >>> paged_kv_accept(k_cache, v_cache, table, lens, accepted, accepted_lens=n)
    >>> lens += n

Every length, position and page table entry stays on the device, so a step can be
captured into a CUDA graph and replayed with new ones.  Extension: the reference
has no cache.

The cache: ``k_cache`` / ``v_cache`` float16 or bfloat16 [num_pages, kv_heads,
page_size, head_dim], any page / head / slot strides (a [num_pages, page_size,
kv_heads, head_dim] cache is passed as ``.transpose(1, 2)``; a contiguous
[batch, kv_heads, seq, head_dim] cache has page_size seq and the table
``arange(batch)[:, None]``).  page_size is a power of two from 8 up or any size
from 64 up, head_dim one of SUPPORTED_HEAD_DIMS_PAGED.  ``page_table`` int32
[batch, max_pages] and ``cache_lens`` int32 [batch]: slot s of sequence b is row
s % page_size of page page_table[b, s // page_size].  Keys are stored rotated.

These values are not known to the host, so the kernels check them: lengths are
clamped to the table's capacity; a page outside the cache is not written and reads
as zeros; a token whose position lies outside the rotation tables is not appended,
and its attention row is zero.
"""
import torch

from . import RDNAttentionError, _last_error, _lib_handle

SUPPORTED_HEAD_DIMS_PAGED = tuple(range(32, 257, 32))
MAX_TREE_TOKENS = 256
MAX_ACCEPTED_TOKENS = 256

_DTYPE_CODES = {torch.float16: 0, torch.bfloat16: 1}


def _tensor(name, t, dtype, device, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on the same device as k_cache")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")


def _optional_int32(name, t, device, shape):
    """Address of a contiguous int32 tensor, or None."""
    if t is None:
        return None
    _tensor(name, t, torch.int32, device, shape)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous - call .contiguous() first")
    return t.data_ptr()


def _cache_args(k_cache, v_cache, page_table, cache_lens):
    """Checks what every call shares; returns (device, dtype code, cache shape, batch, max_pages)."""
    if not isinstance(k_cache, torch.Tensor) or not isinstance(v_cache, torch.Tensor):
        raise TypeError("k_cache and v_cache must be torch.Tensors")
    device, dtype = k_cache.device, k_cache.dtype
    if not k_cache.is_cuda:
        raise ValueError("k_cache must be on a CUDA device")
    code = _DTYPE_CODES.get(dtype)
    if code is None:
        raise ValueError(f"k_cache must be float16 or bfloat16, got {dtype}")
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be 4D [num_pages, kv_heads, page_size, head_dim], got {tuple(k_cache.shape)}")
    shape = tuple(k_cache.shape)
    _tensor("v_cache", v_cache, dtype, device, shape)
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("k_cache and v_cache must have a contiguous head_dim axis")
    if shape[3] not in SUPPORTED_HEAD_DIMS_PAGED:
        raise RDNAttentionError(f"head_dim {shape[3]} not supported (allowed: {list(SUPPORTED_HEAD_DIMS_PAGED)})")
    _tensor("page_table", page_table, torch.int32, device)
    if page_table.dim() != 2 or page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table must be 2D [batch, max_pages] with contiguous rows")
    batch, max_pages = page_table.shape
    _tensor("cache_lens", cache_lens, torch.int32, device, (batch,))
    if not cache_lens.is_contiguous():
        raise ValueError("cache_lens must be contiguous - call .contiguous() first")
    return device, code, shape, batch, max_pages


def _rope_tables(rot_cos, rot_sin, device, head_dim):
    """(cos address, sin address, rows), or (None, None, 0)."""
    if rot_cos is None and rot_sin is None:
        return None, None, 0
    if rot_cos is None or rot_sin is None:
        raise ValueError("pass both rot_cos and rot_sin, or neither")
    for name, t in (("rot_cos", rot_cos), ("rot_sin", rot_sin)):
        _tensor(name, t, torch.float32, device)
        if t.dim() != 2 or t.shape[1] != head_dim // 2:
            raise ValueError(f"{name} must be 2D [positions, head_dim // 2 = {head_dim // 2}], got {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous - call .contiguous() first")
    if rot_cos.shape != rot_sin.shape:
        raise ValueError("rot_cos and rot_sin shapes must match")
    return rot_cos.data_ptr(), rot_sin.data_ptr(), rot_cos.shape[0]


def _new_rows(name, t, k_cache, batch, heads):
    """Checks a [batch, heads, tokens, head_dim] tensor of the cache's type; returns its number of tokens."""
    _tensor(name, t, k_cache.dtype, k_cache.device)
    if t.dim() != 4 or t.shape[0] != batch or t.shape[3] != k_cache.shape[3] or heads and t.shape[1] != heads:
        raise ValueError(f"{name} must be 4D [batch = {batch}, heads, tokens, head_dim = {k_cache.shape[3]}]"
                         f"{f' with {heads} heads' if heads else ''}, got {tuple(t.shape)}")
    if t.stride(3) != 1:
        raise ValueError(f"{name} must have a contiguous head_dim axis")
    return t.shape[2]


def _call(who, device, fn, *args):
    """Runs a library call on `device`'s current stream, with `device` current."""
    if device.index is None or device.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise RDNAttentionError(f"{who} failed: {_last_error()}")


def paged_kv_append(key, value, k_cache, v_cache, page_table, cache_lens, new_lens=None, positions=None,
                    rot_cos=None, rot_sin=None):
    """Writes new tokens into a paged cache, in place.  key / value: [batch, kv_heads,
    tokens, head_dim] of the cache's type (any strides, head_dim contiguous).  Token
    t < new_lens[b] (int32 [batch]; None: all) of sequence b goes to slot
    cache_lens[b] + t, its key turned to positions[b, t] (int32 [batch, tokens];
    None: cache_lens[b] + t) by the float32 [positions, head_dim // 2] tables
    rot_cos / rot_sin as interleaved pairs (None: stored as it is).  No two tokens
    may go to the same row.  Returns (k_cache, v_cache)."""
    device, code, (num_pages, heads, page_size, head_dim), batch, max_pages = _cache_args(
        k_cache, v_cache, page_table, cache_lens)
    tokens = _new_rows("key", key, k_cache, batch, heads)
    if _new_rows("value", value, k_cache, batch, heads) != tokens:
        raise ValueError(f"key and value shapes must match: K={tuple(key.shape)}, V={tuple(value.shape)}")
    new_p = _optional_int32("new_lens", new_lens, device, (batch,))
    pos_p = _optional_int32("positions", positions, device, (batch, tokens))
    cos_p, sin_p, rows = _rope_tables(rot_cos, rot_sin, device, head_dim)
    if batch == 0 or tokens == 0:
        return k_cache, v_cache
    ks, vs, kc, vc = key.stride(), value.stride(), k_cache.stride(), v_cache.stride()
    _call("paged_kv_append", device, _lib_handle().rdna_paged_kv_append,
          key.data_ptr(), value.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(),
          cache_lens.data_ptr(), new_p, pos_p, cos_p, sin_p, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
          kc[0], kc[1], kc[2], vc[0], vc[1], vc[2], page_table.stride(0), batch, heads, tokens, head_dim,
          num_pages, page_size, max_pages, rows, code)
    return k_cache, v_cache


def flash_attn_paged(query, k_cache, v_cache, page_table, cache_lens, new_lens=None, tree_mask=None, positions=None,
                     rot_cos=None, rot_sin=None, window_size: int = -1, scale=None, out=None):
    """Attention of new tokens over a paged cache that holds them already (slots
    cache_lens[b] + t, see paged_kv_append).  query: [batch, heads, tokens,
    head_dim] of the cache's type (any strides, head_dim contiguous; heads an exact
    multiple of the cache's); rot_cos / rot_sin turn it in the kernel to
    positions[b, t] (None: cache_lens[b] + t).

    Without ``tree_mask`` the tokens are a chain: token t sees slots 0 ..
    cache_lens[b] + t (one decode step, or a chunk of a prompt).  ``tree_mask``, bool
    [batch or 1, tokens, tokens] or [tokens, tokens], at most MAX_TREE_TOKENS tokens:
    token t sees every slot below cache_lens[b] and the drafted tokens u <
    new_lens[b] with mask[b, t, u] (itself only if the mask says so).  window_size >
    0: a token sees only the newest window_size of these; its drafted tokens count
    first, in index order (parents before children).  Drafted tokens below
    new_lens[b] must hold finite values; slots behind them may hold anything.

    Softmax scale: ``scale``, None for 1/sqrt(head_dim).  Returns ``out`` (or a new
    tensor) shaped like query; rows t >= new_lens[b] and rows that see nothing are
    zero."""
    device, code, (num_pages, kv_heads, page_size, head_dim), batch, max_pages = _cache_args(
        k_cache, v_cache, page_table, cache_lens)
    tokens = _new_rows("query", query, k_cache, batch, 0)
    heads = query.shape[1]
    if kv_heads == 0 or heads == 0 or heads % kv_heads != 0:
        raise ValueError(f"Q heads ({heads}) must be a multiple of the cache's heads ({kv_heads})")
    new_p = _optional_int32("new_lens", new_lens, device, (batch,))
    pos_p = _optional_int32("positions", positions, device, (batch, tokens))
    cos_p, sin_p, rows = _rope_tables(rot_cos, rot_sin, device, head_dim)
    mask_p, mask_b, mask_t = None, 0, 0
    if tree_mask is not None:
        _tensor("tree_mask", tree_mask, torch.bool, device)
        shape = tuple(tree_mask.shape)
        if shape not in ((tokens, tokens), (1, tokens, tokens), (batch, tokens, tokens)):
            raise ValueError(f"tree_mask must be [batch or 1, tokens, tokens] or [tokens, tokens], got {shape}")
        if tokens > MAX_TREE_TOKENS:
            raise ValueError(f"tree_mask takes at most {MAX_TREE_TOKENS} tokens, got {tokens}")
        if tokens > 1 and (tree_mask.stride(-1) != 1 or tree_mask.stride(-2) < 0):
            raise ValueError("tree_mask must have contiguous rows")
        mask_p = tree_mask.data_ptr()
        mask_t = tree_mask.stride(-2)
        mask_b = tree_mask.stride(0) if len(shape) == 3 and shape[0] > 1 else 0
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=device)
    else:
        _tensor("out", out, query.dtype, device, tuple(query.shape))
        if out.stride(3) != 1:
            raise ValueError("out must have a contiguous head_dim axis")
    if batch == 0 or tokens == 0:
        return out
    lib = _lib_handle()
    ws_bytes = lib.rdna_attention_paged_workspace_size(batch, heads, kv_heads, tokens, head_dim, page_size, max_pages)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    qs, kc, vc, os_ = query.stride(), k_cache.stride(), v_cache.stride(), out.stride()
    _call("flash_attn_paged", device, lib.rdna_attention_forward_paged,
          query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), page_table.data_ptr(),
          cache_lens.data_ptr(), new_p, mask_p, pos_p, cos_p, sin_p, qs[0], qs[1], qs[2], kc[0], kc[1], kc[2],
          vc[0], vc[1], vc[2], os_[0], os_[1], os_[2], mask_b, mask_t, page_table.stride(0), batch, heads, kv_heads,
          tokens, head_dim, num_pages, page_size, max_pages, rows,
          head_dim ** -0.5 if scale is None else float(scale), int(window_size), code, ws.data_ptr(), ws_bytes)
    return out


def paged_kv_accept(k_cache, v_cache, page_table, cache_lens, accepted, accepted_lens=None):
    """Moves the accepted drafted tokens to the front of the drafted slots, in place:
    slot cache_lens[b] + i takes the row of slot cache_lens[b] + accepted[b, i] for i <
    accepted_lens[b] (int32 [batch]; None: all), all rows as they were before the call
    (the same token twice is fine).  accepted: int32 [batch, n], n at most
    MAX_ACCEPTED_TOKENS; a negative entry, or one behind the page table, moves nothing.
    The drafted slots' pages must belong to one sequence only.  Returns (k_cache,
    v_cache)."""
    device, code, (num_pages, heads, page_size, head_dim), batch, max_pages = _cache_args(
        k_cache, v_cache, page_table, cache_lens)
    _tensor("accepted", accepted, torch.int32, device)
    if accepted.dim() != 2 or accepted.shape[0] != batch or not accepted.is_contiguous():
        raise ValueError(f"accepted must be contiguous [batch = {batch}, n], got {tuple(accepted.shape)}")
    n = accepted.shape[1]
    if n > MAX_ACCEPTED_TOKENS:
        raise ValueError(f"at most {MAX_ACCEPTED_TOKENS} accepted tokens, got {n}")
    lens_p = _optional_int32("accepted_lens", accepted_lens, device, (batch,))
    if batch == 0 or n == 0:
        return k_cache, v_cache
    kc, vc = k_cache.stride(), v_cache.stride()
    _call("paged_kv_accept", device, _lib_handle().rdna_paged_kv_accept,
          k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(), cache_lens.data_ptr(), accepted.data_ptr(),
          lens_p, kc[0], kc[1], kc[2], vc[0], vc[1], vc[2], page_table.stride(0), batch, heads, head_dim, num_pages,
          page_size, max_pages, n, code)
    return k_cache, v_cache
