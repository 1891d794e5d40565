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
page_size, head_dim], page / head / slot strides positive multiples of 16 bytes,
page and slot strides below 2**31 elements (a [num_pages, page_size, kv_heads,
head_dim] cache is passed as ``.transpose(1, 2)``; a contiguous [batch, kv_heads,
seq, head_dim] cache has page_size seq and the table ``arange(batch)[:, None]``).
page_size is a power of two from 8 up or any size from 64 up, head_dim one of
SUPPORTED_HEAD_DIMS_PAGED.  ``page_table`` int32
[batch, max_pages] and ``cache_lens`` int32 [batch]: slot s of sequence b is row
s % page_size of page page_table[b, s // page_size].  Keys are stored rotated.
A single sequence is attended to faster through a table no wider than it needs
(up to 11000 slots with 8 kv_heads, 18000 with 4 or fewer), ``page_table[:, :n]``: the host, which chooses between
two forms, knows the table's width and not the length.

These values are not known to the host, so the kernels check them: lengths are
clamped to the table's capacity; a page outside the cache is not written and reads
as zeros; a token whose position lies outside the rotation tables is not appended,
and its attention row is zero.
"""
import functools
import struct

from . import RDNAttentionError, _last_error, _lib_handle

SUPPORTED_HEAD_DIMS_PAGED = tuple(range(32, 257, 32))
MAX_TREE_TOKENS = 256
MAX_ACCEPTED_TOKENS = 256

# torch and what depends on it: importing the package needs no torch, the first call loads it
torch = _raw_stream = _DTYPE_CODES = None
_HEAD_DIMS = frozenset(SUPPORTED_HEAD_DIMS_PAGED)

# rdna_paged_cache and the argument structs that start with one (include/rdnattention.h).
# One pack per call: converting the arguments one by one would take longer than the
# smaller kernels.
_CACHE = "4Q7q6IiI"
_APPEND = struct.Struct("=" + _CACHE + "6Q6q2I")
_ATTENTION = struct.Struct("=" + _CACHE + "9Q8q3IifI")
_ACCEPT = struct.Struct("=" + _CACHE + "2Q2I")


def _load_torch():
    global torch, _raw_stream, _DTYPE_CODES
    import torch as module

    try:  # the stream's handle without a Stream object (2 us less per call)
        from torch._C import _cuda_getCurrentRawStream as raw_stream
    except ImportError:
        def raw_stream(index):
            return module.cuda.current_stream(index).cuda_stream

    _raw_stream = raw_stream
    _DTYPE_CODES = {module.float16: 0, module.bfloat16: 1}
    torch = module  # last: another thread's call may run as soon as it is set


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
    """Address of a contiguous int32 tensor, or 0."""
    if t is None:
        return 0
    if (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.device == device and t.shape == shape
            and t.is_contiguous()):
        return t.data_ptr()
    _tensor(name, t, torch.int32, device, shape)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous - call .contiguous() first")
    return t.data_ptr()


def _check_cache(k_cache, v_cache, page_table, cache_lens):
    """Raises what is wrong with the cache's tensors."""
    if not isinstance(k_cache, torch.Tensor) or not isinstance(v_cache, torch.Tensor):
        raise TypeError("k_cache and v_cache must be torch.Tensors")
    device, dtype = k_cache.device, k_cache.dtype
    if not k_cache.is_cuda:
        raise ValueError("k_cache must be on a CUDA device")
    if dtype not in _DTYPE_CODES:
        raise ValueError(f"k_cache must be float16 or bfloat16, got {dtype}")
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be 4D [num_pages, kv_heads, page_size, head_dim], got {tuple(k_cache.shape)}")
    _tensor("v_cache", v_cache, dtype, device, tuple(k_cache.shape))
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("k_cache and v_cache must have a contiguous head_dim axis")
    if k_cache.shape[3] not in _HEAD_DIMS:
        raise RDNAttentionError(
            f"head_dim {k_cache.shape[3]} not supported (allowed: {list(SUPPORTED_HEAD_DIMS_PAGED)})")
    _tensor("page_table", page_table, torch.int32, device)
    if page_table.dim() != 2 or page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table must be 2D [batch, max_pages] with contiguous rows")
    _tensor("cache_lens", cache_lens, torch.int32, device, (page_table.shape[0],))
    if not cache_lens.is_contiguous():
        raise ValueError("cache_lens must be contiguous - call .contiguous() first")


def _cache_args(k_cache, v_cache, page_table, cache_lens):
    """Checks what every call shares; returns (device, shape of the cache, batch, packed rdna_paged_cache values)."""
    try:
        device, dtype, shape, ks = k_cache.device, k_cache.dtype, k_cache.shape, k_cache.stride()
        vs, ts, batch = v_cache.stride(), page_table.stride(), page_table.shape[0]
        max_pages = page_table.shape[1]
        # (all in one expression: these checks are half of a small call)
        good = (device.type == "cuda" and dtype in _DTYPE_CODES and len(shape) == 4 and v_cache.dtype is dtype
                and v_cache.device == device and v_cache.shape == shape and ks[3] == 1 and vs[3] == 1
                and shape[3] in _HEAD_DIMS and page_table.dtype is torch.int32 and page_table.device == device
                and len(ts) == 2 and (ts[1] == 1 or max_pages <= 1) and cache_lens.dtype is torch.int32
                and cache_lens.device == device and cache_lens.shape == (batch,) and cache_lens.is_contiguous())
    except (AttributeError, IndexError, TypeError):
        good = False
    if not good:
        _check_cache(k_cache, v_cache, page_table, cache_lens)
        raise ValueError("unsupported cache tensors")
    return device, shape, batch, (
        k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(), cache_lens.data_ptr(), ks[0], ks[1], ks[2],
        vs[0], vs[1], vs[2], ts[0], batch, shape[1], shape[3], shape[0], shape[2], max_pages, _DTYPE_CODES[dtype], 0)


def _rope_tables(rot_cos, rot_sin, device, head_dim):
    """(cos address, sin address, rows), or (0, 0, 0)."""
    if rot_cos is None and rot_sin is None:
        return 0, 0, 0
    if rot_cos is None or rot_sin is None:
        raise ValueError("pass both rot_cos and rot_sin, or neither")
    if isinstance(rot_cos, torch.Tensor) and isinstance(rot_sin, torch.Tensor):
        shape = rot_cos.shape
        if (rot_cos.dtype is torch.float32 and rot_sin.dtype is torch.float32 and rot_cos.device == device
                and rot_sin.device == device and len(shape) == 2 and rot_sin.shape == shape
                and shape[0] > 0 and shape[1] == head_dim // 2 and rot_cos.is_contiguous() and rot_sin.is_contiguous()):
            return rot_cos.data_ptr(), rot_sin.data_ptr(), shape[0]
    for name, t in (("rot_cos", rot_cos), ("rot_sin", rot_sin)):
        _tensor(name, t, torch.float32, device)
        if t.dim() != 2 or t.shape[1] != head_dim // 2:
            raise ValueError(f"{name} must be 2D [positions, head_dim // 2 = {head_dim // 2}], got {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous - call .contiguous() first")
    if rot_cos.shape != rot_sin.shape:
        raise ValueError("rot_cos and rot_sin shapes must match")
    if rot_cos.shape[0] == 0:
        raise ValueError("rot_cos and rot_sin have no rows")
    return rot_cos.data_ptr(), rot_sin.data_ptr(), rot_cos.shape[0]


def _new_rows(name, t, k_cache, batch, heads, head_dim):
    """Checks a [batch, heads, tokens, head_dim] tensor of the cache's type; returns (tokens, strides)."""
    if isinstance(t, torch.Tensor) and t.dtype is k_cache.dtype and t.device == k_cache.device:
        shape, stride = t.shape, t.stride()
        if (len(shape) == 4 and shape[0] == batch and shape[3] == head_dim and (heads == 0 or shape[1] == heads)
                and stride[3] == 1):
            return shape[2], stride
    _tensor(name, t, k_cache.dtype, k_cache.device)
    if t.dim() != 4 or t.shape[0] != batch or t.shape[3] != head_dim or heads and t.shape[1] != heads:
        raise ValueError(f"{name} must be 4D [batch = {batch}, heads, tokens, head_dim = {head_dim}]"
                         f"{f' with {heads} heads' if heads else ''}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must have a contiguous head_dim axis")


@functools.lru_cache(maxsize=1024)
def _workspace_elements(device_index, *sizes):
    """Workspace of an attention call, in 2-byte elements."""
    with torch.cuda.device(device_index):
        return (_lib_handle().rdna_attention_paged_workspace_size(*sizes) + 1) // 2


def _call(who, device, fn, args):
    """Runs a library call on `device`'s current stream, with `device` current."""
    if device.index == torch.cuda.current_device():
        rc = fn(args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(args, _raw_stream(device.index))
    if rc != 0:
        raise RDNAttentionError(f"{who} failed: {_last_error()}")


def paged_kv_append(key, value, k_cache, v_cache, page_table, cache_lens, new_lens=None, positions=None,
                    rot_cos=None, rot_sin=None):
    """Writes new tokens into a paged cache, in place.  key / value: [batch, kv_heads,
    tokens, head_dim] of the cache's type (head_dim contiguous, the other strides
    positive multiples of 16 bytes).  Token
    t < new_lens[b] (int32 [batch]; None: all) of sequence b goes to slot
    cache_lens[b] + t, its key turned to positions[b, t] (int32 [batch, tokens];
    None: cache_lens[b] + t) by the float32 [positions, head_dim // 2] tables
    rot_cos / rot_sin as interleaved pairs (None: stored as it is).  No two tokens
    may go to the same row.  Returns (k_cache, v_cache)."""
    if torch is None:
        _load_torch()
    device, (_, heads, _, head_dim), batch, cache = _cache_args(k_cache, v_cache, page_table, cache_lens)
    tokens, ks = _new_rows("key", key, k_cache, batch, heads, head_dim)
    value_tokens, vs = _new_rows("value", value, k_cache, batch, heads, head_dim)
    if value_tokens != tokens:
        raise ValueError(f"key and value shapes must match: K={tuple(key.shape)}, V={tuple(value.shape)}")
    new_p = _optional_int32("new_lens", new_lens, device, (batch,))
    pos_p = _optional_int32("positions", positions, device, (batch, tokens))
    cos_p, sin_p, rows = _rope_tables(rot_cos, rot_sin, device, head_dim)
    if batch == 0 or tokens == 0:
        return k_cache, v_cache
    _call("paged_kv_append", device, _lib_handle().rdna_paged_kv_append,
          _APPEND.pack(*cache, key.data_ptr(), value.data_ptr(), new_p, pos_p, cos_p, sin_p, ks[0], ks[1], ks[2],
                       vs[0], vs[1], vs[2], tokens, rows))
    return k_cache, v_cache


def flash_attn_paged(query, k_cache, v_cache, page_table, cache_lens, new_lens=None, tree_mask=None, positions=None,
                     rot_cos=None, rot_sin=None, window_size: int = -1, scale=None, out=None):
    """Attention of new tokens over a paged cache that holds them already (slots
    cache_lens[b] + t, see paged_kv_append).  query: [batch, heads, tokens,
    head_dim] of the cache's type (strides as for paged_kv_append; heads an exact
    multiple of the cache's); rot_cos / rot_sin turn it in the kernel to
    positions[b, t] (None: cache_lens[b] + t).

    Without ``tree_mask`` the tokens are a chain: token t sees slots 0 ..
    cache_lens[b] + t (one decode step, or a chunk of a prompt).  ``tree_mask``, bool
    [batch or 1, tokens, tokens] or [tokens, tokens], at most MAX_TREE_TOKENS tokens:
    token t sees every slot below cache_lens[b] and the drafted tokens u <
    new_lens[b] with mask[b, t, u] (itself only if the mask says so).  window_size >
    0: a token sees only the newest window_size of these; its drafted tokens count
    first, in index order (parents before children).  (Tokens are counted, positions are
    not compared: for masks of a token and its ancestors at positions cache_lens[b] +
    depth both are the same.)  Drafted tokens below
    new_lens[b] must hold finite values; slots behind them, and context slots that no
    token's window reaches, may hold anything.  At most 262144 rows (tokens * heads /
    kv_heads) per sequence, 65536 above head_dim 128.

    Softmax scale: ``scale``, None for 1/sqrt(head_dim).  Returns ``out`` (or a new
    tensor; it must not share memory with query) shaped like query; rows t >= new_lens[b] and rows that see nothing are
    zero."""
    if torch is None:
        _load_torch()
    device, (_, kv_heads, page_size, head_dim), batch, cache = _cache_args(k_cache, v_cache, page_table, cache_lens)
    tokens, qs = _new_rows("query", query, k_cache, batch, 0, head_dim)
    heads = query.shape[1]
    if kv_heads == 0 or heads == 0 or heads % kv_heads != 0:
        raise ValueError(f"Q heads ({heads}) must be a multiple of the cache's heads ({kv_heads})")
    new_p = _optional_int32("new_lens", new_lens, device, (batch,))
    pos_p = _optional_int32("positions", positions, device, (batch, tokens))
    cos_p, sin_p, rows = _rope_tables(rot_cos, rot_sin, device, head_dim)
    mask_p = mask_b = mask_t = 0
    if tree_mask is not None:
        _tensor("tree_mask", tree_mask, torch.bool, device)
        shape = tree_mask.shape
        if shape not in ((tokens, tokens), (1, tokens, tokens), (batch, tokens, tokens)):
            raise ValueError(f"tree_mask must be [batch or 1, tokens, tokens] or [tokens, tokens], got {tuple(shape)}")
        if tokens > MAX_TREE_TOKENS:
            raise ValueError(f"tree_mask takes at most {MAX_TREE_TOKENS} tokens, got {tokens}")
        ms = tree_mask.stride()
        if tokens > 1 and (ms[-1] != 1 or ms[-2] < 0):
            raise ValueError("tree_mask must have contiguous rows")
        mask_p, mask_t = tree_mask.data_ptr(), ms[-2]
        mask_b = ms[0] if len(shape) == 3 and shape[0] > 1 else 0
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    else:
        _tensor("out", out, query.dtype, device, tuple(query.shape))
        if out.stride(3) != 1:
            raise ValueError("out must have a contiguous head_dim axis")
        if out.data_ptr() == query.data_ptr() and out.numel():
            raise ValueError("out must not share memory with query")
    if batch == 0 or tokens == 0:
        return out
    ws = query.new_empty(_workspace_elements(device.index, batch, heads, kv_heads, tokens, head_dim, page_size, cache[-3]))
    os_ = out.stride()
    _call("flash_attn_paged", device, _lib_handle().rdna_attention_forward_paged,
          _ATTENTION.pack(*cache, query.data_ptr(), out.data_ptr(), new_p, mask_p, pos_p, cos_p, sin_p, ws.data_ptr(),
                          2 * ws.numel(), qs[0], qs[1], qs[2], os_[0], os_[1], os_[2], mask_b, mask_t, heads, tokens,
                          rows, max(-1, min(int(window_size), 2**31 - 1)), head_dim ** -0.5 if scale is None else float(scale), 0))
    return out


def paged_kv_accept(k_cache, v_cache, page_table, cache_lens, accepted, accepted_lens=None):
    """Moves the accepted drafted tokens to the front of the drafted slots, in place:
    slot cache_lens[b] + i takes the row of slot cache_lens[b] + accepted[b, i] for i <
    accepted_lens[b] (int32 [batch]; None: all), all rows as they were before the call
    (the same token twice is fine).  accepted: int32 [batch, n], n at most
    MAX_ACCEPTED_TOKENS; a negative entry, or one behind the page table, moves nothing.
    The drafted slots' pages must belong to one sequence only.  Returns (k_cache,
    v_cache)."""
    if torch is None:
        _load_torch()
    device, _, batch, cache = _cache_args(k_cache, v_cache, page_table, cache_lens)
    _tensor("accepted", accepted, torch.int32, device)
    if accepted.dim() != 2 or accepted.shape[0] != batch or not accepted.is_contiguous():
        raise ValueError(f"accepted must be contiguous [batch = {batch}, n], got {tuple(accepted.shape)}")
    n = accepted.shape[1]
    if n > MAX_ACCEPTED_TOKENS:
        raise ValueError(f"at most {MAX_ACCEPTED_TOKENS} accepted tokens, got {n}")
    lens_p = _optional_int32("accepted_lens", accepted_lens, device, (batch,))
    if batch == 0 or n == 0:
        return k_cache, v_cache
    _call("paged_kv_accept", device, _lib_handle().rdna_paged_kv_accept,
          _ACCEPT.pack(*cache, accepted.data_ptr(), lens_p, n, 0))
    return k_cache, v_cache
