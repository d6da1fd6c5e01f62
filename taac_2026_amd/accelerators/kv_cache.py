"""A cache of keys and values in 4 or 8 bits, and softmax attention of new tokens over it: the counterpart of
:func:`gated_delta_rule_step` for models that attend, beside :func:`flash_attention` for whole histories.

The cache is a pool of pages of ``page_tokens`` tokens; a table names the pages of every sample's history, in order. Of 32 consecutive features of a
token's head the values are stored as codes times one power of two, the least with ``max |x| < 7 * 2^e`` (4 bits, e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6) or ``< 464 * 2^e``
(8 bits, e4m3), rounded to nearest even, so that each is off by half a step at most.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass, field

import torch

from taac_2026_amd import _native
from taac_2026_amd.accelerators.head_rope import MAX_COUNT, strides_of, token_major
from taac_2026_amd.accelerators.tensor_validation import require_cuda_tensors, require_inference, require_no_tangents, require_same_dtype

CACHED_WIDTHS = (32, 64, 128)
_CHUNK = 16
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


@functools.lru_cache(maxsize=64)
def _record_bytes(head_dim: int, bits: int) -> int:
    return _native.load_library().taac_kv_cache_bytes(1, 1, _CHUNK, head_dim, bits)


@dataclass(frozen=True, eq=False)
class KVCache:
    """A pool of pages (:func:`empty_kv_cache`). ``data``: uint8 (pages, heads, page_tokens / 16, bytes of 16 tokens), the library's own layout."""

    data: torch.Tensor
    head_dim: int
    bits: int
    pages: int = field(init=False)
    heads: int = field(init=False)
    page_tokens: int = field(init=False)

    def __post_init__(self) -> None:
        data = self.data
        if data.ndim != 4 or data.dtype != torch.uint8 or not data.is_contiguous() or data.shape[3] != _record_bytes(self.head_dim, self.bits):
            raise ValueError("KVCache expects data as made by empty_kv_cache")
        for name, value in (("pages", data.shape[0]), ("heads", data.shape[1]), ("page_tokens", data.shape[2] * _CHUNK)):
            object.__setattr__(self, name, value)


def empty_kv_cache(pages: int, heads: int, head_dim: int, *, bits: int = 4, page_tokens: int = 64, device: torch.device | str) -> KVCache:
    """A pool of ``pages`` pages that hold ``page_tokens`` tokens (a power of two, at least 16) of ``heads`` key heads of 32, 64 or 128 features, in 4 or 8 bits
    and one byte per 32 features."""
    if bits not in (4, 8):
        raise ValueError(f"a cache has 4 or 8 bits, got {bits}")
    if head_dim not in CACHED_WIDTHS:
        raise ValueError(f"a cached head has {', '.join(map(str, CACHED_WIDTHS))} features, got {head_dim}")
    if page_tokens < _CHUNK or page_tokens > 1 << 16 or page_tokens & (page_tokens - 1) != 0:
        raise ValueError(f"a page has a power of two of tokens, {_CHUNK} to 65536, got {page_tokens}")
    if pages < 0 or heads <= 0:
        raise ValueError("a cache needs heads and a number of pages that is not negative")
    data = torch.zeros(pages, heads, page_tokens // _CHUNK, _record_bytes(head_dim, bits), dtype=torch.uint8, device=device)
    return KVCache(data, int(head_dim), int(bits))


def _check_pages(name: str, pages: torch.Tensor, batch: int) -> None:
    if pages.ndim != 2 or pages.shape[0] != batch or pages.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} expects a table of pages (batch, pages of a sample) in int32 or int64")
    if pages.stride(1) != 1 and pages.shape[1] > 1:
        raise ValueError(f"{name} expects a table whose rows are contiguous")


def _check_counts(name: str, batch: int, tokens: int, pages: torch.Tensor) -> None:
    if batch > MAX_COUNT or tokens > MAX_COUNT or pages.shape[1] > MAX_COUNT:
        raise RuntimeError(f"hip {name} is built for samples, tokens and pages of a sample of at most 2^31 - 1")


def _integers(name: str, what: str, t: torch.Tensor, batch: int) -> torch.Tensor:
    if t.shape != (batch,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} {what} must hold one int32 or int64 per sample")
    return t if t.stride(0) == 1 else t.contiguous()


def _lengths(name: str, what: str, t: torch.Tensor | None, batch: int) -> torch.Tensor | None:
    if t is None:
        return None
    t = _integers(name, what, t, batch)
    # more than the library's 32 bits count as the most that they hold
    return t if t.dtype == torch.int32 else t.clamp(-1, 2**31 - 1).to(torch.int32)


def _pool(cache: KVCache, pages: torch.Tensor) -> tuple:
    return (cache.data.data_ptr(), cache.pages, cache.heads, cache.page_tokens, cache.head_dim, cache.bits, pages.data_ptr(),
            int(pages.dtype == torch.int64), pages.stride(0), pages.shape[1])


def _in_place(t: torch.Tensor, size: int) -> torch.Tensor:
    """``t`` where the library can read it (contiguous rows at 16-byte addresses), else a copy."""
    batch, head, token, feature = t.stride()
    if feature == 1 and (batch | head | token) * size % 16 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def kv_cache_write(
    cache: KVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    pages: torch.Tensor,
    starts: torch.Tensor | None = None,
    *,
    lengths: torch.Tensor | None = None,
) -> None:
    """Quantises ``k, v (batch, key heads, tokens, width)`` into the cache: token t of a sample to position ``starts[b] + t`` (without starts: t), i.e. into page
    ``pages[b, position // page_tokens]``. ``lengths (batch,)``: the tokens that a sample really has; the others are not read. A token whose page is not in the
    table or not in the pool (-1 for a padded sample) is left out, and all of a sample whose start is negative. Places that two tokens of a call share hold a mixture of both afterwards.

    float32, bfloat16 or float16. A token whose key or value, in a head, has a NaN or an infinity is stored as NaN there. Forward only."""
    name = "kv_cache_write"
    if k.ndim != 4 or k.shape != v.shape:
        raise ValueError(f"{name} expects k and v of one shape (batch, heads, tokens, width)")
    if k.shape[1] != cache.heads or k.shape[3] != cache.head_dim:
        raise ValueError(f"{name} expects {cache.heads} heads of {cache.head_dim} features, got {k.shape[1]} of {k.shape[3]}")
    if k.dtype != v.dtype:
        require_same_dtype(f"{name} k, v", k, v)
    batch, _, tokens, _ = k.shape
    _check_pages(name, pages, batch)
    starts = None if starts is None else _integers(name, "starts", starts, batch)
    lengths = _lengths(name, "lengths", lengths, batch)
    require_no_tangents(f"hip {name}", k, v)
    require_cuda_tensors(f"hip {name}", cache.data, k, v, pages, starts, lengths)
    require_inference(f"hip {name}", k, v)
    if k.dtype not in _DTYPES:
        raise RuntimeError(f"hip {name} does not support dtype {k.dtype}")
    _check_counts(name, batch, tokens, pages)
    size = k.element_size()
    k, v = _in_place(k, size), _in_place(v, size)
    with _native.on_device(k.device):
        status = _native.load_library().taac_kv_cache_write(
            *_pool(cache, pages), k.data_ptr(), v.data_ptr(), _native.ptr(starts), int(starts is not None and starts.dtype == torch.int64),
            _native.ptr(lengths), batch, tokens, strides_of(k), strides_of(v), _native.dtype_code(k.dtype), _native.current_stream(k.device))
    _native.check(status, name)
    torch.autograd.graph.increment_version(cache.data)


def kv_cache_read(
    cache: KVCache,
    pages: torch.Tensor,
    starts: torch.Tensor | None,
    tokens: int,
    *,
    lengths: torch.Tensor | None = None,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)`` of ``tokens`` positions from ``starts[b]`` on (without starts: 0), the values that the codes stand for, as (batch, key heads, tokens, width) in memory
    order (batch, tokens, heads, width). Positions at or beyond ``lengths[b]`` tokens, and those in no page of the pool, are zeros, as is all of a sample whose start is negative. Exact in bfloat16 and
    float32; in float16 where it reaches."""
    name = "kv_cache_read"
    batch = pages.shape[0] if pages.ndim == 2 else -1
    _check_pages(name, pages, batch)
    if int(tokens) < 0:
        raise ValueError(f"{name} needs a number of tokens that is not negative")
    starts = None if starts is None else _integers(name, "starts", starts, batch)
    lengths = _lengths(name, "lengths", lengths, batch)
    require_cuda_tensors(f"hip {name}", cache.data, pages, starts, lengths)
    if dtype not in _DTYPES:
        raise RuntimeError(f"hip {name} does not support dtype {dtype}")
    _check_counts(name, batch, int(tokens), pages)
    k, v = (token_major((batch, cache.heads, int(tokens), cache.head_dim), cache.data, dtype) for _ in range(2))
    with _native.on_device(k.device):
        status = _native.load_library().taac_kv_cache_read(
            *_pool(cache, pages), k.data_ptr(), v.data_ptr(), _native.ptr(starts), int(starts is not None and starts.dtype == torch.int64),
            _native.ptr(lengths), batch, int(tokens), strides_of(k), strides_of(v), _native.dtype_code(dtype), _native.current_stream(k.device))
    _native.check(status, name)
    return k, v


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch: int, heads: int, key_heads: int, tokens: int, width: int, bits: int, table_tokens: int) -> int:
    return _native.load_library().taac_cached_attention_workspace_bytes(batch, heads, key_heads, tokens, width, bits, table_tokens)


def cached_attention(
    q: torch.Tensor,
    cache: KVCache,
    pages: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float | None = None,
    query_lengths: torch.Tensor | None = None,
    window: int | None = None,
) -> torch.Tensor:
    """``softmax(scale q k^T) v`` of the new tokens ``q (batch, heads, tokens, width)`` over the cached keys and values -> the shape of q, in memory order (batch,
    tokens, heads, width). Query heads are a multiple of the cache's; consecutive ones share a key head. ``scale`` defaults to ``width ** -0.5``.

    ``lengths (batch,)`` counts the tokens that a sample has in the cache, the new ones among them: they are written first (:func:`kv_cache_write`), and query t
    of a sample with n of them stands at position ``lengths[b] - n + t``, where n is ``query_lengths[b]``, else ``tokens``. It sees the positions up to its own, with
    ``window`` the last ``window`` of them, itself included. Queries at or beyond ``query_lengths[b]`` and queries that see nothing get zeros, positions in no page of
    the pool are not seen.

    bfloat16 or float16 queries. They, keys and values enter exactly; scores, statistics and sums are float32; probabilities enter the product with 24 bits where a
    key head has up to four rows (query heads that share it times tokens; two of float16), else with 16; the output is rounded once. A NaN or an infinity in a cached token reaches the queries that see it, and no others.
    Forward only."""
    name = "cached_attention"
    if q.ndim != 4:
        raise ValueError(f"{name} expects q with shape (batch, heads, tokens, width)")
    batch, heads, tokens, width = q.shape
    if width != cache.head_dim or heads == 0 or heads % cache.heads != 0:
        raise ValueError(f"{name} expects a multiple of {cache.heads} heads of {cache.head_dim} features, got {heads} of {width}")
    _check_pages(name, pages, batch)
    lengths = _lengths(name, "lengths", lengths, batch)
    query_lengths = _lengths(name, "query_lengths", query_lengths, batch)
    if window is not None and (int(window) != window or window <= 0):
        raise ValueError(f"{name} window must be a number of tokens above zero")
    require_no_tangents(f"hip {name}", q)
    require_cuda_tensors(f"hip {name}", q, cache.data, pages, lengths, query_lengths)
    require_inference(f"hip {name}", q)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"hip {name} does not support dtype {q.dtype}")
    _check_counts(name, batch, tokens, pages)
    q = _in_place(q, 2)
    out = token_major(q.shape, q)
    bytes_needed = _workspace_bytes(batch, heads, cache.heads, tokens, width, cache.bits, pages.shape[1] * cache.page_tokens if cache.pages > 0 else 0)
    workspace = q.new_empty(bytes_needed, dtype=torch.uint8) if bytes_needed > 0 else None
    with _native.on_device(q.device):
        status = _native.load_library().taac_cached_attention_fwd(
            q.data_ptr(), out.data_ptr(), *_pool(cache, pages), lengths.data_ptr(), _native.ptr(query_lengths),
            0 if window is None else min(int(window), 2**31 - 1), width ** -0.5 if scale is None else float(scale), _native.ptr(workspace), max(bytes_needed, 0),
            batch, heads, tokens, strides_of(q), strides_of(out), _native.dtype_code(q.dtype), _native.current_stream(q.device))
    _native.check(status, name)
    return out


__all__ = ["KVCache", "cached_attention", "empty_kv_cache", "kv_cache_read", "kv_cache_write"]
