"""The paged cache's argument checks (no GPU): the C entries refuse before touching the device."""
import ctypes

import pytest
import torch

from sta import _lib as L
from sta import paged


def cache_args(**kw):
    c = L.PagedCacheArgs()
    for f in ("k", "v", "table", "lens", "weights"):
        setattr(c, f, 256)  # non-null placeholders: these calls return before any device work
    c.dtype, c.d, c.n_pages, c.n_kv_heads, c.page_size, c.batch, c.table_width = 1, 128, 100, 8, 16, 4, 50
    c.table_stride, c.weights_stride_p, c.weights_stride_h = 50, 128, 16
    for x in "kv":
        setattr(c, f"{x}_stride_n", 128)
        setattr(c, f"{x}_stride_h", 128 * 16)
        setattr(c, f"{x}_stride_p", 128 * 16 * 8)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def decode_args(**kw):
    a = L.PagedDecodeArgs(256, 32 * 128, 128, 256, 32, 256, 1.0, 1.0, 0.088)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def evict_args(**kw):
    a = L.PagedEvictArgs(64, 4, 4, 256, 4, 4, 256, 4096)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def refused(rc, text):
    assert rc in (1, 2), rc
    assert text in L.lib().sta_last_error(), L.lib().sta_last_error()


BAD_CACHE = [
    (dict(k=None), b"null"), (dict(lens=None), b"null"), (dict(d=96), b"64 or 128"),
    (dict(dtype=2), b"f32 or bf16"), (dict(n_pages=0), b"sizes"), (dict(batch=-1), b"sizes"),
    (dict(page_size=0), b"page_size"), (dict(page_size=65537), b"page_size"),
    (dict(table_width=1 << 27), b"2^31"), (dict(k_stride_n=129), b"16 bytes"),
    (dict(v_stride_h=4), b"16 bytes"), (dict(k=264), b"16-byte"),
]


@pytest.mark.parametrize("kw,text", BAD_CACHE)
def test_bad_caches_are_refused(kw, text):
    lib, c = L.lib(), cache_args(**kw)
    app = L.PagedAppendArgs(256, 128, 128, 128, 256, 128, 128, 128, 1, None, 4096)
    refused(lib.sta_paged_append(ctypes.byref(c), ctypes.byref(app), None), text)
    assert lib.sta_paged_decode_workspace_bytes(ctypes.byref(c), ctypes.byref(decode_args())) == 0
    refused(lib.sta_paged_decode(ctypes.byref(c), ctypes.byref(decode_args()), None, 0, None), text)
    refused(lib.sta_paged_evict(ctypes.byref(c), ctypes.byref(evict_args()), None, 0, None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(inv_freq=None), b"null"),
    (dict(n_heads=12), b"multiple"), (dict(n_heads=0), b"multiple"),
    (dict(chunk_size=100, local_window=100), b"chunk_size"), (dict(chunk_size=-1), b"chunk_size"),
    (dict(chunk_size=320, local_window=32), b"64"),
    (dict(chunk_size=320, local_window=64, pos_scale=0.5), b"pos_scale"),
])
def test_bad_decodes_are_refused(kw, text):
    lib, c, a = L.lib(), cache_args(), decode_args(**kw)
    refused(lib.sta_paged_decode(ctypes.byref(c), ctypes.byref(a), None, 0, None), text)


def test_decode_weights_need_a_cache_with_weights_and_a_workspace():
    lib = L.lib()
    refused(lib.sta_paged_decode(ctypes.byref(cache_args(weights=None)),
                                 ctypes.byref(decode_args(weights_out=512)), None, 0, None), b"weights")
    c, a = cache_args(), decode_args()
    need = lib.sta_paged_decode_workspace_bytes(ctypes.byref(c), ctypes.byref(a))
    assert need > 0
    assert lib.sta_paged_decode(ctypes.byref(c), ctypes.byref(a), 256, need - 1, None) == 5
    assert lib.sta_paged_decode(ctypes.byref(c), ctypes.byref(a), None, need, None) == 5


@pytest.mark.parametrize("kw,text", [
    (dict(budget=0), b"budget"), (dict(n_global=-1), b"n_global"), (dict(n_global=60, n_local=5), b"n_global"),
    (dict(table_out=None), b"null"), (dict(kept=None), b"null"), (dict(table_out_width=3), b"no room"),
    (dict(table_out_width=0), b"empty"), (dict(lens_out=256 + 4), b"overlaps"), (dict(lens_out=256), b"overlaps"),
])
def test_bad_evictions_are_refused(kw, text):
    lib, c, a = L.lib(), cache_args(), evict_args(**kw)
    refused(lib.sta_paged_evict(ctypes.byref(c), ctypes.byref(a), 256, 1 << 30, None), text)


def test_evict_needs_weights_and_a_workspace():
    lib = L.lib()
    refused(lib.sta_paged_evict(ctypes.byref(cache_args(weights=None)), ctypes.byref(evict_args()), 256, 1 << 30, None),
            b"weights")
    c, a = cache_args(), evict_args()
    need = lib.sta_paged_evict_workspace_bytes(ctypes.byref(c), ctypes.byref(a))
    assert need > 0 and lib.sta_paged_evict(ctypes.byref(c), ctypes.byref(a), 256, need - 1, None) == 5


def test_bad_appends_are_refused():
    lib, c = L.lib(), cache_args()

    def app(n=1, k=256, lens_out=4096):
        return ctypes.byref(L.PagedAppendArgs(k, 128, 128, 128, 256, 128, 128, 128, n, None, lens_out))

    refused(lib.sta_paged_append(ctypes.byref(c), None, None), b"null")
    refused(lib.sta_paged_append(ctypes.byref(c), app(n=-1), None), b"bad n")
    refused(lib.sta_paged_append(ctypes.byref(c), app(k=None), None), b"null")
    refused(lib.sta_paged_append(ctypes.byref(c), app(lens_out=None), None), b"null")
    refused(lib.sta_paged_append(ctypes.byref(c), app(lens_out=256 + 4), None), b"overlaps")


@pytest.mark.parametrize("offset", [-4, 4])
def test_lengths_must_not_overlap_part_of_the_counts(offset):
    lib, c = L.lib(), cache_args()
    assert c.batch > 1
    a = L.PagedAppendArgs(256, 128, 128, 128, 256, 128, 128, 128, 1, 4096, 4096 + offset)
    refused(lib.sta_paged_append(ctypes.byref(c), ctypes.byref(a), None), b"overlaps counts")


def test_an_empty_batch_is_a_no_op():
    lib, c = L.lib(), cache_args(batch=0)
    app = L.PagedAppendArgs(256, 128, 128, 128, 256, 128, 128, 128, 1, None, 4096)
    assert lib.sta_paged_append(ctypes.byref(c), ctypes.byref(app), None) == 0
    assert lib.sta_paged_decode(ctypes.byref(c), ctypes.byref(decode_args()), None, 0, None) == 0
    assert lib.sta_paged_evict(ctypes.byref(c), ctypes.byref(evict_args()), None, 0, None) == 0


def test_cpu_tensors_are_refused():
    k = torch.zeros((4, 2, 16, 64))
    with pytest.raises(ValueError):
        paged.PagedCache(k, k, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_struct_layouts_match_header_order():
    import os
    import re
    here = os.path.dirname(os.path.abspath(__file__))
    src = open(os.path.join(os.path.dirname(here), "include", "sta.h")).read()
    for cname, cls in (("sta_paged_cache", L.PagedCacheArgs), ("sta_paged_append_args", L.PagedAppendArgs),
                       ("sta_paged_decode_args", L.PagedDecodeArgs), ("sta_paged_evict_args", L.PagedEvictArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), src, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        assert [f for f, _ in cls._fields_] == re.findall(r"\**\s*([A-Za-z_0-9]+)\s*;", body), cname
