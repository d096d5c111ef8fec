"""The paged cache's host side: what a caller could break or overlap (no GPU)."""
import ctypes

import pytest
import torch

from sta import _lib as L
from sta import paged
from test_paged_cpu import cache_args, decode_args, evict_args, refused


@pytest.mark.parametrize("name", ["k", "v", "table", "lens", "weights", "device"])
def test_the_tensors_of_a_cache_cannot_be_exchanged(name):
    """The addresses are taken once: another tensor under the same name would go unread, and the
    one that the kernels go on using would be freed."""
    cache = paged.PagedCache.__new__(paged.PagedCache)
    cache._tensors = tuple(torch.zeros(i + 1) for i in range(5)) + (torch.device("cpu"),)
    with pytest.raises(AttributeError):
        setattr(cache, name, torch.zeros(9))
    assert cache.k.numel() == 1 and cache.lens.numel() == 4 and cache.device.type == "cpu"


def append_args():
    return L.PagedAppendArgs(256, 128, 128, 128, 256, 128, 128, 128, 1, None, 4096)


@pytest.mark.parametrize("name,text", [
    ("k_stride_p", b"K / V are written"), ("k_stride_h", b"K / V are written"), ("k_stride_n", b"K / V are written"),
    ("v_stride_p", b"K / V are written"), ("v_stride_h", b"K / V are written"), ("v_stride_n", b"K / V are written"),
    ("weights_stride_p", b"weights are written"), ("weights_stride_h", b"weights are written"),
])
def test_what_is_written_has_no_stride_of_zero(name, text):
    """A broadcast pool (heads or pages expanded) would take the rows of several slots in one place."""
    lib, c = L.lib(), ctypes.byref(cache_args(**{name: 0}))
    refused(lib.sta_paged_append(c, ctypes.byref(append_args()), None), text)
    refused(lib.sta_paged_evict(c, ctypes.byref(evict_args()), 256, 1 << 30, None), text)
    read = lib.sta_paged_decode(c, ctypes.byref(decode_args()), None, 0, None)
    assert read == 5  # only read: nothing but the workspace is missing
    if name[0] == "w":
        refused(lib.sta_paged_decode(c, ctypes.byref(decode_args(weights_out=1 << 30)), None, 0, None), text)


def test_a_dimension_of_one_may_have_a_stride_of_zero():
    lib = L.lib()
    c = cache_args(n_kv_heads=1, k_stride_h=0, v_stride_h=0, weights_stride_h=0, batch=0)
    assert lib.sta_paged_append(ctypes.byref(c), ctypes.byref(append_args()), None) == 0
    assert lib.sta_paged_evict(ctypes.byref(c), ctypes.byref(evict_args()), None, 0, None) == 0


# weights of 100 pages, 8 heads, 16 slots at address 4096; strides of pages and heads, where weights_out begins
@pytest.mark.parametrize("strides,offset,overlaps", [
    ((128, 16), 0, False),                # the weights themselves
    ((128, 16), 1, True), ((128, 16), -1, True), ((128, 16), 16, True), ((128, 16), -128, True),
    ((128, 16), 100 * 128 - 1, True), ((128, 16), 100 * 128, False), ((128, 16), -100 * 128, False),
    ((256, 16), 128, False),              # pages of both in turn
    ((256, 16), 127, True), ((256, 16), 256 + 128, False), ((256, 16), 256, True),
    ((256, 32), 16, False), ((256, 32), 15, True), ((256, 32), -16, False),  # heads of both in turn
    ((16, 1600), 16, True), ((16, 3200), 1600, False),  # heads first
    ((24, 2400), 8, True),                # gaps between the pages, too short for another array
    ((32, 3200), 16, False), ((32, 3200), -17, True),
])
def test_weights_out_is_the_weights_or_apart_from_them(strides, offset, overlaps):
    lib = L.lib()
    at = 1 << 20
    c = cache_args(weights=at, weights_stride_p=strides[0], weights_stride_h=strides[1])
    a = decode_args(weights_out=at + 4 * offset)
    places = {p * strides[0] + h * strides[1] + r for p in range(100) for h in range(8) for r in range(16)}
    assert overlaps == (offset != 0 and any(x + offset in places for x in places))
    need = lib.sta_paged_decode_workspace_bytes(ctypes.byref(c), ctypes.byref(a))
    if overlaps:
        assert need == 0
        refused(lib.sta_paged_decode(ctypes.byref(c), ctypes.byref(a), None, 0, None), b"overlaps the weights")
    else:
        assert need > 0 and lib.sta_paged_decode(ctypes.byref(c), ctypes.byref(a), None, 0, None) == 5


def test_frequencies_elsewhere_are_refused_in_a_capture(monkeypatch):
    """Copying them waits for the copy, which a capture does not survive."""
    dev = torch.device("meta")
    cache = paged.PagedCache.__new__(paged.PagedCache)
    pool = torch.zeros((3, 2, 4, 64), device=dev)
    cache._tensors = (pool, pool, None, None, None, dev)
    cache._args, cache._sizes = cache_args(batch=2, d=64, n_kv_heads=2), {}
    q = torch.zeros((2, 4, 64), device=dev)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ValueError, match="inv_freq must lie on"):
        paged.decode(q, cache, paged.Geometry(torch.ones(32)))
    with pytest.raises(ValueError, match="head_dim/2"):  # there: the next check
        paged.decode(q, cache, paged.Geometry(torch.ones(31, device=dev)))


def test_the_package_imports_where_torch_has_no_cuda(monkeypatch):
    """torch built without CUDA lacks the bindings that the calls use; importing needs none of them."""
    import importlib.util
    import sys
    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        monkeypatch.delattr(torch._C, name)
    spec = importlib.util.spec_from_file_location("sta._paged_without_cuda", paged.__file__)
    module = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(sys.modules, spec.name, module)
    spec.loader.exec_module(module)
    with pytest.raises(ValueError):
        module.PagedCache(torch.zeros((4, 2, 16, 64)), None, None, None)
