"""Refusals of the per-head norm with rotation, of the cache and of the attention over it that need no GPU, and the table's own arithmetic."""

from __future__ import annotations

import ctypes
import itertools
import re

import pytest
import torch

from taac_2026_amd import _native
from taac_2026_amd.api import KVCache, cached_attention, empty_kv_cache, head_norm_rope, kv_cache_read, kv_cache_write, rotary_table


def test_rotary_table_refuses():
    for arguments in ((-1, 32), (4, 0), (4, 31), (4, -2)):
        with pytest.raises(ValueError, match="even number"):
            rotary_table(*arguments)
    for options in ({"base": 0.0}, {"base": float("inf")}, {"factor": -1.0}, {"factor": float("nan")}):
        with pytest.raises(ValueError, match="above zero"):
            rotary_table(4, 32, **options)
    for options in ({"trained_places": 0}, {"trained_places": 8, "turns": (3.0, 3.0)}):
        with pytest.raises(ValueError, match="ascending"):
            rotary_table(4, 32, factor=2.0, **options)
    table = rotary_table(5, 8)
    assert table.shape == (5, 4, 2) and table.dtype == torch.float32 and table.is_contiguous() and torch.equal(table[0], torch.tensor([[1.0, 0.0]] * 4))
    assert rotary_table(0, 8).shape == (0, 4, 2)
    assert torch.equal(rotary_table(5, 8, factor=3.0, trained_places=10**9), table)  # every frequency turns often enough to stay


def test_head_norm_rope_refuses():
    q, k, w, table = torch.zeros(2, 4, 3, 32), torch.zeros(2, 2, 3, 32), torch.ones(32), rotary_table(8, 16)
    for a, b in ((q[0], k), (q, k[0])):
        with pytest.raises(ValueError, match="shape \\(batch, heads"):
            head_norm_rope(a, b, w, w)
    for a, b in ((q[:1], k), (q, k[:, :, :2]), (q, k[..., :16]), (q[:, :0], k), (q[..., :0], k[..., :0])):
        with pytest.raises(ValueError, match="matching batch"):
            head_norm_rope(a, b, w, w)
    with pytest.raises(ValueError, match="same dtype"):
        head_norm_rope(q, k.bfloat16(), w, w)
    with pytest.raises(ValueError, match="both norm weights"):
        head_norm_rope(q, k, w)
    with pytest.raises(ValueError, match="or both"):
        head_norm_rope(q, k)
    with pytest.raises(ValueError, match="one value per feature"):
        head_norm_rope(q, k, w, w[:16])
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            head_norm_rope(q, k, w, w, eps=eps)
    place = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="not both"):
        head_norm_rope(q, k, w, w, table=table, starts=place, positions=place)
    with pytest.raises(ValueError, match="come with a table"):
        head_norm_rope(q, k, w, w, starts=place)
    with pytest.raises(ValueError, match="int32 or int64"):
        head_norm_rope(q, k, w, w, table=table, starts=place.float())
    with pytest.raises(ValueError, match="one position per sample"):
        head_norm_rope(q, k, w, w, table=table, starts=place[:1])
    for shape in ((2,), (3, 2), (1, 3), (2, 3, 1)):
        with pytest.raises(ValueError, match="shape \\(tokens,\\)"):
            head_norm_rope(q, k, w, w, table=table, positions=torch.zeros(shape, dtype=torch.int64))
    for wrong in (rotary_table(8, 34), table[..., :1], table[0], table[:, :0]):
        with pytest.raises(ValueError, match="rotated / 2, 2"):
            head_norm_rope(q, k, w, w, table=wrong)
    for wrong in (table.double(), table.transpose(0, 1)):
        with pytest.raises(ValueError, match="contiguous float32"):
            head_norm_rope(q, k, w, w, table=wrong)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        head_norm_rope(q, k, w, w, table=table, starts=place)


def test_cache_refuses():
    for options, match in (({"bits": 3}, "4 or 8"), ({"page_tokens": 24}, "power of two"), ({"page_tokens": 8}, "power of two"), ({"page_tokens": 1 << 17}, "power of two")):
        with pytest.raises(ValueError, match=match):
            empty_kv_cache(1, 1, 32, device="cpu", **options)
    with pytest.raises(ValueError, match="features"):
        empty_kv_cache(1, 1, 48, device="cpu")
    for pages, heads in ((-1, 1), (1, 0)):
        with pytest.raises(ValueError, match="needs heads"):
            empty_kv_cache(pages, heads, 32, device="cpu")
    cache = empty_kv_cache(6, 2, 64, bits=8, page_tokens=32, device="cpu")
    assert (cache.pages, cache.heads, cache.page_tokens, cache.head_dim, cache.bits) == (6, 2, 32, 64, 8)
    assert cache.data.numel() == 6 * 2 * 2 * 32 * (64 + 2) and (cache.data == 0).all()
    k, pages = torch.zeros(3, 2, 5, 64), torch.zeros(3, 2, dtype=torch.int32)
    write = lambda k=k, v=k, pages=pages, *rest, **options: kv_cache_write(cache, k, v, pages, *rest, **options)  # noqa: E731
    for a, b in ((k[0], k[0]), (k, k[:, :, :4])):
        with pytest.raises(ValueError, match="one shape"):
            write(a, b)
    for x in (k[:, :1], k[..., :32]):
        with pytest.raises(ValueError, match="2 heads of 64 features"):
            write(x, x)
    with pytest.raises(ValueError, match="same dtype"):
        write(k, k.half())
    for wrong in (pages[0], pages[:2], pages.float(), pages.bool()):
        with pytest.raises(ValueError, match="table of pages"):
            write(pages=wrong)
    with pytest.raises(ValueError, match="rows are contiguous"):
        write(pages=torch.zeros(2, 3, dtype=torch.int32).t())
    for wrong in (torch.zeros(2, dtype=torch.int32), torch.zeros(3), torch.zeros(3, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="starts"):
            kv_cache_write(cache, k, k, pages, wrong)
        with pytest.raises(ValueError, match="lengths"):
            kv_cache_write(cache, k, k, pages, lengths=wrong)
        with pytest.raises(ValueError, match="starts"):
            kv_cache_read(cache, pages, wrong, 4)
    for data in (cache.data[..., :-1], cache.data.int(), cache.data[0], cache.data[:, ::2]):
        with pytest.raises(ValueError, match="empty_kv_cache"):
            kv_cache_write(KVCache(data, 64, 8), k, k, pages)
    with pytest.raises(ValueError, match="not negative"):
        kv_cache_read(cache, pages, None, -1)
    with pytest.raises(ValueError, match="table of pages"):
        kv_cache_read(cache, pages[0], None, 1)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        write()
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        kv_cache_read(cache, pages, None, 4)


def test_cached_attention_refuses():
    cache = empty_kv_cache(6, 2, 64, page_tokens=32, device="cpu")
    q, pages, lengths = torch.zeros(3, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="shape \\(batch, heads"):
        cached_attention(q[0], cache, pages, lengths)
    for wrong in (q[:, :3], q[:, :0], q[..., :32]):
        with pytest.raises(ValueError, match="multiple of 2 heads"):
            cached_attention(wrong, cache, pages, lengths)
    with pytest.raises(ValueError, match="table of pages"):
        cached_attention(q, cache, pages[:1], lengths)
    for wrong in (lengths[:2], lengths.float()):
        with pytest.raises(ValueError, match="lengths"):
            cached_attention(q, cache, pages, wrong)
        with pytest.raises(ValueError, match="query_lengths"):
            cached_attention(q, cache, pages, lengths, query_lengths=wrong)
    for window in (0, -1, 1.5):
        with pytest.raises(ValueError, match="window"):
            cached_attention(q, cache, pages, lengths, window=window)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        cached_attention(q, cache, pages, lengths)


def test_a_cache_is_itself():
    """Compared and hashed as one object, not by its tensor."""
    a, b = (empty_kv_cache(1, 1, 32, device="cpu") for _ in range(2))
    assert a == a and a != b and len({a, b, a}) == 2


def test_rope_entry_points_check_on_the_host():
    library = _native.load_library()
    fake = ctypes.c_void_p(256)
    invalid, unsupported, ok = _native.TAAC_ERR_INVALID_VALUE, _native.TAAC_ERR_UNSUPPORTED, _native.TAAC_OK
    s = (ctypes.c_int64 * 3)(96, 32, 32)

    def both(**kw):
        a = dict(q=fake, B=1, H=2, Hk=1, T=3, d=32, rotary=16, qs=s, w=fake, kw=fake, eps=1e-6, table=fake, places=8, positions=None, ps=None, dtype=_native.TAAC_BF16)
        a.update(kw)
        rest = (a["w"], a["kw"], a["eps"], a["table"], a["places"], a["positions"], 0, a["ps"], 0, 0, a["dtype"], None)
        sizes = (a["B"], a["H"], a["Hk"], a["T"], a["d"], a["rotary"])
        forward = library.taac_head_norm_rope_fwd(a["q"], fake, fake, fake, *sizes, a["qs"], s, s, s, *rest)
        backward = library.taac_head_norm_rope_bwd(a["q"], fake, fake, fake, fake, fake, fake, fake, fake, 1 << 20, *sizes, a["qs"], s, s, s, s, s, *rest)
        assert forward == backward
        return forward

    assert both(B=-1) == invalid and both(T=-1) == invalid and both(H=0) == invalid and both(Hk=0) == invalid and both(d=0) == invalid
    assert both(d=513) == unsupported and both(H=(1 << 20) + 1) == unsupported
    assert both(rotary=15) == invalid and both(rotary=34) == invalid and both(rotary=-2) == invalid and b"rotated" in library.taac_last_error()
    assert both(rotary=0) == invalid and both(table=None) == invalid and both(places=-1) == invalid
    assert both(places=1 << 31) == unsupported and b"2^31 - 1" in library.taac_last_error()
    assert both(w=None) == invalid and both(kw=None) == invalid and b"both norm weights" in library.taac_last_error()
    assert both(dtype=7) == invalid and both(eps=-1.0) == invalid and both(qs=None) == invalid and both(q=None) == invalid
    assert both(positions=fake) == invalid and b"positions" in library.taac_last_error()
    assert both(table=ctypes.c_void_p(258)) == invalid
    # without rows and weights there is nothing to launch
    assert both(B=0, w=None, kw=None) == ok and both(T=0, w=None, kw=None) == ok
    size = library.taac_head_norm_rope_bwd_workspace_floats
    assert size(2, 4, 4, 100, 32) == 2 * 32 * 25 and size(0, 4, 4, 100, 32) == 0 and size(1, 0, 1, 1, 32) == -1 and size(1, 1, 1, 1, 513) == -1
    arguments = [fake, fake, fake, fake, fake, fake, fake, fake, fake, 10, 2, 4, 4, 100, 32, 16, s, s, s, s, s, s, fake, fake, 1e-6, fake, 8, None, 0, None, 0, 0, 1, None]
    assert library.taac_head_norm_rope_bwd(*arguments) == invalid and b"workspace" in library.taac_last_error()
    arguments[6] = None
    assert library.taac_head_norm_rope_bwd(*arguments) == invalid and b"gradients" in library.taac_last_error()


def test_cache_entry_points_check_on_the_host():
    library = _native.load_library()
    fake, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)
    invalid, unsupported, ok = _native.TAAC_ERR_INVALID_VALUE, _native.TAAC_ERR_UNSUPPORTED, _native.TAAC_OK
    size = library.taac_kv_cache_bytes
    assert size(3, 2, 64, 32, 4) == 3 * 2 * 64 * (32 + 2) and size(3, 2, 64, 128, 8) == 3 * 2 * 64 * (256 + 8) and size(0, 1, 16, 32, 4) == 0
    for wrong in ((-1, 2, 64, 32, 4), (3, 0, 64, 32, 4), (3, 2, 48, 32, 4), (3, 2, 8, 32, 4), (3, 2, 64, 96, 4), (3, 2, 64, 32, 6)):
        assert size(*wrong) == -1
    strides = lambda *x: (ctypes.c_int64 * 3)(*x)  # noqa: E731

    def both(**kw):
        a = dict(cache=fake, pages=4, heads=2, page=16, d=32, bits=4, table=fake, table_pages=2, k=fake, B=1, T=3, ks=strides(192, 32, 64), dtype=_native.TAAC_BF16)
        a.update(kw)
        arguments = (a["cache"], a["pages"], a["heads"], a["page"], a["d"], a["bits"], a["table"], 0, 2, a["table_pages"], a["k"], fake, None, 0, None, a["B"], a["T"],
                     a["ks"], strides(192, 32, 64), a["dtype"], None)
        write, read = library.taac_kv_cache_write(*arguments), library.taac_kv_cache_read(*arguments)
        assert write == read
        return write

    assert both(B=-1) == invalid and both(T=-1) == invalid and both(pages=-1) == invalid and both(heads=0) == invalid and both(table_pages=-1) == invalid
    assert both(d=48) == unsupported and both(bits=2) == unsupported and both(page=17) == unsupported and both(page=1 << 17) == unsupported
    assert both(heads=(1 << 16) + 1) == unsupported
    assert both(cache=None) == invalid and both(cache=odd) == invalid and both(table=None) == invalid and both(k=None) == invalid and both(k=odd) == invalid
    assert both(ks=None) == invalid and both(ks=strides(192, 33, 64)) == invalid and b"16 bytes" in library.taac_last_error()
    assert both(dtype=9) == invalid
    assert both(B=0) == ok and both(T=0) == ok

    def attend(**kw):
        a = dict(q=fake, o=fake, cache=fake, pages=4, heads=2, page=16, d=32, bits=4, table=fake, table_pages=2, lengths=fake, window=0, ws=None, bytes=0, B=1, H=4, T=1,
                 qs=strides(128, 32, 128), os=strides(128, 32, 128), dtype=_native.TAAC_BF16)
        a.update(kw)
        return library.taac_cached_attention_fwd(
            a["q"], a["o"], a["cache"], a["pages"], a["heads"], a["page"], a["d"], a["bits"], a["table"], 0, a["table_pages"], a["table_pages"], a["lengths"], None,
            a["window"], 1.0, a["ws"], a["bytes"], a["B"], a["H"], a["T"], a["qs"], a["os"], a["dtype"], None)

    assert attend(H=3) == invalid and attend(H=0) == invalid and attend(B=-1) == invalid and attend(T=-1) == invalid
    assert attend(d=16) == unsupported and attend(bits=5) == unsupported and attend(page=20) == unsupported
    assert attend(dtype=_native.TAAC_F32) == invalid and attend(window=-1) == invalid
    assert attend(qs=None) == invalid and attend(qs=strides(128, 36, 128)) == invalid and attend(os=strides(128, 34, 128)) == invalid
    assert attend(q=None) == invalid and attend(o=None) == invalid and attend(lengths=None) == invalid and attend(q=odd) == invalid and attend(o=ctypes.c_void_p(260)) == invalid
    assert attend(table_pages=1 << 27) == unsupported and b"2^30" in library.taac_last_error()
    assert attend(H=1 << 21, T=32) == unsupported and b"queries" in library.taac_last_error()
    assert attend(heads=1 << 16, H=1 << 16, T=1 << 13) == unsupported and b"workgroups" in library.taac_last_error()
    assert attend(B=0) == ok and attend(T=0) == ok
    need = library.taac_cached_attention_workspace_bytes(1, 4, 2, 1, 32, 4, 1 << 16)
    assert need > 0 and attend(table_pages=1 << 12, ws=fake, bytes=need - 1) == invalid and b"workspace" in library.taac_last_error()
    assert attend(table_pages=1 << 12, ws=odd, bytes=need) == invalid
    for d in (32, 64, 128):  # queries of either type find room in what is asked for
        for group, bits in itertools.product((1, 2, 3, 4, 5, 16, 17), (4, 8)):
            need = library.taac_cached_attention_workspace_bytes(1, 8 * group, 8, 1, d, bits, 1 << 16)
            asked = []
            for dtype in (_native.TAAC_BF16, _native.TAAC_F16):
                assert attend(heads=8, H=8 * group, d=d, bits=bits, table_pages=1 << 12, dtype=dtype) == invalid
                asked.append(int(re.search(rb"must hold (\d+) bytes", library.taac_last_error()).group(1)))
            assert need == max(asked)
    assert library.taac_cached_attention_workspace_bytes(1024, 8, 8, 1, 32, 4, 512) == 0  # enough samples to fill the card
    assert library.taac_cached_attention_workspace_bytes(1, 3, 2, 1, 32, 4, 512) == -1 and library.taac_cached_attention_workspace_bytes(1, 2, 2, 1, 32, 6, 512) == -1


def test_a_table_of_no_places_is_one():
    """Its pointer is null, and every position lies outside it."""
    library = _native.load_library()
    fake, s = ctypes.c_void_p(256), (ctypes.c_int64 * 3)(96, 32, 32)

    def forward(tokens, rotary, table, places):
        return library.taac_head_norm_rope_fwd(fake, fake, fake, fake, 1, 2, 1, tokens, 32, rotary, s, s, s, s, fake, fake, 1e-6, table, places, None, 0, None, 0, 0,
                                               _native.TAAC_BF16, None)

    assert forward(0, 16, None, 0) == _native.TAAC_OK
    assert forward(0, 16, None, 1) == _native.TAAC_ERR_INVALID_VALUE and forward(0, 0, fake, 0) == _native.TAAC_ERR_INVALID_VALUE


def test_tangents_are_refused():
    """Whatever carries one; without any, a level of forward-mode differentiation changes nothing."""
    from torch.autograd import forward_ad

    q, w, table = torch.zeros(2, 4, 3, 32), torch.ones(32), rotary_table(8, 16)
    cache, pages, lengths = empty_kv_cache(6, 4, 32, page_tokens=16, device="cpu"), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    calls = (
        (lambda q, k, wq, wk, table: head_norm_rope(q, k, wq, wk, table=table), (q, q, w, w, table)),
        (lambda k, v: kv_cache_write(cache, k, v, pages), (q, q)),
        (lambda q: cached_attention(q, cache, pages, lengths), (q.bfloat16(),)),
    )
    with forward_ad.dual_level():
        for call, arguments in calls:
            with pytest.raises(RuntimeError, match="CUDA tensors"):
                call(*arguments)
            for i, t in enumerate(arguments):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*arguments[:i], forward_ad.make_dual(t, torch.ones_like(t)), *arguments[i + 1:])
