"""Serving from a paged key/value cache: prompts as a whole, single tokens, and
sequences that fork, end and are packed together.

The reference generates from no cache (ssalaad/inference/generate.py:1-26);
`DecodeEngine` keeps one dense cache per slot. Here keys and values live in two
pools of pages, [pages, kv_heads, page, head_dim] for one layer or
[layers, pages, kv_heads, page, head_dim], and a table [seqs, cols] int32 names
the page of each run of `page` positions of a sequence (-1: none):

  paged_append             rotary embedding of new tokens, k and v into their pages
  paged_decode_attention   one new token per sequence over its pages
  paged_prompt_attention   chunks of tokens, causal, ragged
  free_pages / fork_pages  sequences that end, and that go on more than once
  compact_pages            the pages in use moved to the lowest numbers

float32, bfloat16 and float16; head_dim 64, 128 or 256; pages of 16 to 1024
positions (a power of two); any number of query heads per key/value head. Every
call runs on torch's current stream, reads lengths, positions and page numbers
on the device (none synchronises) and may be captured into a HIP graph. Page
numbers outside the pool are treated as no page. There is no CPU path and no
gradient (inputs that require one give plain outputs). What free_pages,
fork_pages and compact_pages return shares one allocation a call, their
workspace in it: an output that is kept keeps all of it.

Each function first hands its call to the compiled path (csrc_py/tensorcall.cpp),
which takes arguments that are as the kernels want them; what it leaves is
checked, and laid out anew where needed, here.
"""

from __future__ import annotations

import struct

import torch

from . import _lib

# The C ABI's argument structs: ssl_paged_cache (size, pools, table, dtype) and
# what each call adds to it.
_CACHE = "=17q"
_APPEND = struct.Struct(_CACHE + "16qd5q")
_ATTENTION = struct.Struct(_CACHE + "10qd4q")
_PAGES = struct.Struct(_CACHE + "12q")

_ALIGN = {torch.float32: 4, torch.bfloat16: 8, torch.float16: 8}  # elements of 16 bytes


def _call(name: str, args: bytes, device: torch.device) -> None:
    lib = _lib.load()
    if device.index == torch.cuda.current_device():
        rc = getattr(lib, name)(args, _lib.stream_ptr(device))
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, name)(args, _lib.stream_ptr(device))
    if rc:
        _lib.check(rc, name)


def _on_gpu(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"the paged cache lives on a ROCm GPU device; move {name} there first")
    return t.device


def _ints(t: torch.Tensor, name: str, shape: tuple, device: torch.device) -> torch.Tensor:
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the pools are on {device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    return t if t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if t.dtype is not torch.int32:
        raise TypeError(f"the page table must be int32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"the page table is on {t.device}, the pools are on {device}")
    if t.dim() != 2:
        raise ValueError("the page table must be 2-D, [seqs, cols]")
    s = t.stride()
    if (s[1] != 1 and t.shape[1] > 1) or s[0] < t.shape[1]:
        t = t.contiguous()
    return t


def _rows(t: torch.Tensor, name: str, shape: tuple, like: torch.Tensor) -> torch.Tensor:
    """[tokens, heads, head_dim] with 16-byte rows (a copy where it has none)."""
    if t.dtype is not like.dtype:
        raise TypeError(f"{name} is {t.dtype}, the pools are {like.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, the pools are on {like.device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    s, a = t.stride(), _ALIGN[t.dtype]
    if s[2] != 1 or s[0] % a or s[1] % a or s[0] < 0 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _pools(k: torch.Tensor, v: torch.Tensor, layers: bool) -> tuple:
    """ssl_paged_cache's fields from k to head_dim."""
    _on_gpu(k, "k_pool")
    if k.dtype not in _ALIGN:
        _lib.dtype_code(k.dtype)
    if v.dtype is not k.dtype:
        raise TypeError(f"k_pool is {k.dtype}, v_pool {v.dtype}")
    if v.device != k.device:
        raise ValueError(f"k_pool is on {k.device}, v_pool on {v.device}")
    sh, st = k.shape, k.stride()
    if len(sh) == 4:
        sh, st = (1, *sh), (0, *st)
    elif len(sh) != 5 or not layers:
        raise ValueError("the pools must be [pages, kv_heads, page, head_dim]"
                         + (" or [layers, pages, kv_heads, page, head_dim]" if layers else "")
                         + f", got {tuple(sh)}")
    if v.shape != k.shape or v.stride() != k.stride():
        raise ValueError("k_pool and v_pool must have the same shape and strides")
    if k.numel() == 0:
        raise ValueError("the pools hold no page")
    a = _ALIGN[k.dtype]
    if st[4] != 1 or any(x % a for x in st[:4]) or k.data_ptr() % 16 or v.data_ptr() % 16:
        raise ValueError("the pools must have contiguous features and 16-byte aligned strides")
    return (k.data_ptr(), v.data_ptr(), *st[:4], *sh)


def _grid(table: torch.Tensor) -> tuple:
    """ssl_paged_cache's table fields."""
    return table.data_ptr(), table.stride(0) if table.shape[0] > 1 else table.shape[1], *table.shape


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 table: torch.Tensor, seqs: torch.Tensor, positions: torch.Tensor, *,
                 q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                 eps: float = 1e-6) -> torch.Tensor:
    """Rotate the new tokens' q and k, write k and v into one layer's pages
    (in place) and return the rotated q [tokens, heads, head_dim].

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim]; token t
    belongs to sequence seqs[t] at positions[t] (int32). cos and sin are fp32
    [angles, head_dim / 2], the halves of a head rotated against each other.
    q_norm, k_norm [head_dim]: an RMS norm per head before the rotation. A
    position without an angle gives a zero row; it and one without a page are
    not written. No two tokens may share a place.
    """
    out = _lib.tensorcall().append(q, k, v, cos, sin, k_pool, v_pool, table, seqs, positions,
                                   q_norm, k_norm, eps)
    if out is not None:
        return _lib.completed(out, "ssl_paged_append")
    pools = _pools(k_pool, v_pool, False)
    dev, hd, kv = k_pool.device, pools[10], pools[8]
    if q.dim() != 3:
        raise ValueError("q must be 3-D, [tokens, heads, head_dim]")
    n, heads = q.shape[0], q.shape[1]
    q = _rows(q, "q", (n, heads, hd), k_pool)
    k = _rows(k, "k", (n, kv, hd), k_pool)
    v = _rows(v, "v", (n, kv, hd), k_pool)
    table = _table(table, dev)
    seqs = _ints(seqs, "seqs", (n,), dev)
    positions = _ints(positions, "positions", (n,), dev)
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise TypeError("cos and sin must be float32")
    if cos.dim() != 2 or cos.shape[1] * 2 != hd or sin.shape != cos.shape:
        raise ValueError(f"cos and sin must be [angles, {hd // 2}]")
    if cos.device != dev or sin.device != dev:
        raise ValueError("cos and sin must be on the pools' device")
    if cos.stride(1) != 1 or cos.stride(0) % 4 or cos.data_ptr() % 16:
        cos = cos.clone(memory_format=torch.contiguous_format)
    if sin.stride(1) != 1 or sin.stride(0) % 4 or sin.data_ptr() % 16:
        sin = sin.clone(memory_format=torch.contiguous_format)
    norms = []
    for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if w is not None:
            if w.dtype is not k_pool.dtype:
                raise TypeError(f"{name} is {w.dtype}, the pools are {k_pool.dtype}")
            if w.shape != (hd,) or w.device != dev:
                raise ValueError(f"{name} must be [{hd}] on {dev}")
            if w.stride(0) != 1 or w.data_ptr() % 16:
                w = w.clone(memory_format=torch.contiguous_format)
        norms.append(w)
    out = torch.empty((n, heads, hd), dtype=q.dtype, device=dev)
    if n:
        _call("ssl_paged_append", _APPEND.pack(
            _APPEND.size, *pools, *_grid(table), _lib.dtype_code(q.dtype),
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
            v.data_ptr(), v.stride(0), v.stride(1), cos.data_ptr(), sin.data_ptr(),
            cos.stride(0), sin.stride(0), cos.shape[0], _lib.ptr(norms[0]) or 0,
            _lib.ptr(norms[1]) or 0, eps, seqs.data_ptr(), positions.data_ptr(), out.data_ptr(), n,
            heads), dev)
    return out


def _attention(q, k_pool, v_pool, table, lengths, cu, window, sinks, scale, max_tokens, max_length):
    out = _lib.tensorcall().attention(q, k_pool, v_pool, table, lengths, cu, window, sinks, scale,
                                      max_tokens, max_length)
    if out is not None:
        return _lib.completed(out, "ssl_paged_attention")
    pools = _pools(k_pool, v_pool, False)
    dev, hd = k_pool.device, pools[10]
    if q.dim() != 3:
        raise ValueError("q must be 3-D, [tokens, heads, head_dim]")
    n, heads = q.shape[0], q.shape[1]
    if heads == 0 or heads % pools[8]:
        raise ValueError(f"{heads} query heads over {pools[8]} key/value heads")
    q = _rows(q, "q", (n, heads, hd), k_pool)
    table = _table(table, dev)
    seqs, cols = table.shape
    lengths = _ints(lengths, "lengths", (seqs,), dev)
    if cu is not None:
        cu = _ints(cu, "cu", (seqs + 1,), dev)
    elif n != seqs:
        raise ValueError(f"{n} tokens for {seqs} sequences")
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must be nonnegative")
    reach = cols * pools[9]
    if max_length is None or max_length > reach:
        max_length = reach
    if max_tokens is None or max_tokens > n:
        max_tokens = n
    if max_length < 0 or max_tokens < 0:
        raise ValueError("max_tokens and max_length must be nonnegative")
    out = torch.empty((n, heads, hd), dtype=q.dtype, device=dev)
    if n:
        fields = [_ATTENTION.size, *pools, *_grid(table), _lib.dtype_code(q.dtype), q.data_ptr(),
                  q.stride(0), q.stride(1), out.data_ptr(), lengths.data_ptr(),
                  0 if cu is None else cu.data_ptr(), n, heads, window, sinks,
                  hd ** -0.5 if scale is None else scale, max_tokens, max_length, 0, 0]
        need = _lib.load().ssl_paged_attention_workspace_size(_ATTENTION.pack(*fields))
        if need:
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            fields[-2:] = work.data_ptr(), need
        _call("ssl_paged_attention", _ATTENTION.pack(*fields), dev)
    return out


def paged_decode_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                           table: torch.Tensor, lengths: torch.Tensor, *, window: int = 0,
                           sinks: int = 0, scale: float | None = None,
                           max_length: int | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over one layer's pages.

    q [seqs, heads, head_dim]; lengths [seqs] int32 counts the cached positions,
    the new token's own (the last) among them; length 0 gives zeros. With a
    window the token sees its last `window` positions and the first `sinks`.
    max_length, a bound of the lengths, shapes the launch only. scale defaults
    to head_dim ** -0.5. Returns [seqs, heads, head_dim].
    """
    return _attention(q, k_pool, v_pool, table, lengths, None, window, sinks, scale, 1, max_length)


def paged_prompt_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                           table: torch.Tensor, lengths: torch.Tensor, cu: torch.Tensor, *,
                           window: int = 0, sinks: int = 0, scale: float | None = None,
                           max_tokens: int | None = None,
                           max_length: int | None = None) -> torch.Tensor:
    """Causal attention of chunks of tokens over one layer's pages.

    q [tokens, heads, head_dim]: tokens cu[s] … cu[s + 1] − 1 (cu [seqs + 1]
    int32, ascending from 0) are sequence s's last ones, written into its pages
    before; lengths [seqs] int32 counts them. A token at position p sees the
    positions up to p, with a window the last `window` of them and the first
    `sinks`; one that sees none gives zeros, as do tokens past cu[seqs].
    max_tokens and max_length, bounds of a sequence's tokens and length, shape
    the launch only. Returns [tokens, heads, head_dim].
    """
    if cu is None:
        raise TypeError("cu must be an int32 tensor [seqs + 1]")
    return _attention(q, k_pool, v_pool, table, lengths, cu, window, sinks, scale, max_tokens,
                      max_length)


def _state(table, refs, device):
    table = _table(table, device)
    if refs.dim() != 1 or refs.shape[0] == 0:
        raise ValueError("refs must be 1-D, one count a page")
    refs = _ints(refs, "refs", tuple(refs.shape), device)
    return (table, refs, torch.empty(tuple(table.shape), dtype=torch.int32, device=device),
            torch.empty_like(refs))


def free_pages(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
               seqs: torch.Tensor):
    """End the sequences `seqs` (int32): (table, lengths, refs) with their rows
    -1, their lengths 0 and one reference less for every entry they held. refs
    [pages] int32 counts the entries that name a page; one at 0 is free. A
    sequence named twice ends once; one out of range is passed over. The given
    tensors stay as they are."""
    out = _lib.tensorcall().free(table, lengths, refs, seqs)
    if out is not None:
        return _lib.completed(out, "ssl_pages_free")
    dev = _on_gpu(table, "the page table")
    if seqs.dim() != 1:
        raise ValueError("seqs must be 1-D")
    table, refs, table_out, refs_out = _state(table, refs, dev)
    lengths = _ints(lengths, "lengths", (table.shape[0],), dev)
    seqs = _ints(seqs, "seqs", tuple(seqs.shape), dev)
    lengths_out = torch.empty_like(lengths)
    _call("ssl_pages_free", _PAGES.pack(
        _PAGES.size, 0, 0, 0, 0, 0, 0, 1, refs.shape[0], 1, 16, 64, *_grid(table), 0,
        lengths.data_ptr(), refs.data_ptr(), 0, seqs.data_ptr(), seqs.shape[0],
        table_out.data_ptr(), lengths_out.data_ptr(), refs_out.data_ptr(), 0, 0, 0, 0), dev)
    return table_out, lengths_out, refs_out


def fork_pages(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
               k_pool: torch.Tensor, v_pool: torch.Tensor, src: torch.Tensor,
               dst: torch.Tensor):
    """Let sequence dst[i] (ended, length 0) go on as src[i] does:
    (table, lengths, refs, ok). Whole pages are shared; a partly filled last one
    is copied, in every layer, into the lowest free page (in place in the
    pools); pages that dst's row still names lose that reference. Forks are served in order, all from the state before the call. ok
    [n] bool is False, and nothing changes, where src or dst is out of range,
    dst is not empty or was named before, a page of src is missing, or no page
    is free."""
    out = _lib.tensorcall().fork(table, lengths, refs, k_pool, v_pool, src, dst)
    if out is not None:
        return _lib.completed(out, "ssl_pages_fork")
    pools = _pools(k_pool, v_pool, True)
    dev = k_pool.device
    if src.dim() != 1:
        raise ValueError("src and dst must be 1-D")
    table, refs, table_out, refs_out = _state(table, refs, dev)
    if refs.shape[0] != pools[7]:
        raise ValueError(f"refs counts {refs.shape[0]} pages, the pools hold {pools[7]}")
    lengths = _ints(lengths, "lengths", (table.shape[0],), dev)
    src = _ints(src, "src", tuple(src.shape), dev)
    dst = _ints(dst, "dst", tuple(src.shape), dev)
    n = src.shape[0]
    lengths_out = torch.empty_like(lengths)
    ok = torch.empty(n, dtype=torch.bool, device=dev)
    need = _lib.load().ssl_pages_fork_workspace_size(n)
    work = torch.empty(need, dtype=torch.uint8, device=dev)
    _call("ssl_pages_fork", _PAGES.pack(
        _PAGES.size, *pools, *_grid(table), _lib.dtype_code(k_pool.dtype), lengths.data_ptr(),
        refs.data_ptr(), src.data_ptr(), dst.data_ptr(), n, table_out.data_ptr(),
        lengths_out.data_ptr(), refs_out.data_ptr(), ok.data_ptr(), 0, work.data_ptr(), need), dev)
    return table_out, lengths_out, refs_out, ok


def compact_pages(table: torch.Tensor, refs: torch.Tensor, k_pool: torch.Tensor,
                  v_pool: torch.Tensor):
    """Move the pages in use to the lowest numbers: (table, refs, live). With
    `live` (0-d int32) of them, the i-th used page at or above it moves into the
    i-th free one below it, in every layer (in place in the pools), and the
    table's entries follow. Pages from `live` on are free afterwards."""
    out = _lib.tensorcall().compact(table, refs, k_pool, v_pool)
    if out is not None:
        return _lib.completed(out, "ssl_pages_compact")
    pools = _pools(k_pool, v_pool, True)
    dev = k_pool.device
    table, refs, table_out, refs_out = _state(table, refs, dev)
    if refs.shape[0] != pools[7]:
        raise ValueError(f"refs counts {refs.shape[0]} pages, the pools hold {pools[7]}")
    live = torch.empty((), dtype=torch.int32, device=dev)
    need = _lib.load().ssl_pages_compact_workspace_size(pools[7])
    work = torch.empty(need, dtype=torch.uint8, device=dev)
    _call("ssl_pages_compact", _PAGES.pack(
        _PAGES.size, *pools, *_grid(table), _lib.dtype_code(k_pool.dtype), 0, refs.data_ptr(),
        0, 0, 0, table_out.data_ptr(), 0, refs_out.data_ptr(), 0, live.data_ptr(),
        work.data_ptr(), need), dev)
    return table_out, refs_out, live
