"""The paged key-value cache: calls that the documentation allows and the first set of tests does
not make (needs a B200)."""
import math

import pytest
import torch

import paged_ref as ref
from sta import core, paged
from sta.core import Geometry
from test_gpu_paged import check_decode, inv_freq, on_gpu, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,G", [(64, 2), (64, 12), (128, 4), (128, 12)])
@pytest.mark.parametrize("page,strided", [(16, False), (32, True), (24, False)])  # dense rows, rows of a page, any rows
def test_every_key_of_a_unit_with_a_bad_page_is_nan(D, G, page, strided):
    """The NaN that stands for a bad page's keys is written over the zeros of the copies: in every
    layout of rows all of the sequence's heads see it, call after call."""
    lens, hk = [400, 410, 390, 77], 4
    c = ref.make(lens, hk=hk, D=D, page=page, dtype=torch.bfloat16, seed=201)
    for t in (0, 3, 11):
        c["table"][1, t] = -1
    c["table"][3, 77 // page] = c["k"].shape[0]
    d, cache = on_gpu(c)
    if strided:
        k, v = (torch.zeros(x.shape[:3] + (2, D), dtype=x.dtype, device="cuda")[..., 0, :] for x in (d["k"], d["v"]))
        k.copy_(d["k"])
        v.copy_(d["v"])
        cache = paged.PagedCache(k, v, d["table"], d["lens"])
    q = queries(4, hk * G, D, torch.bfloat16, 202)
    geo = Geometry(inv_freq(D).cuda())
    for _ in range(20):
        out = paged.decode(q.cuda(), cache, geo)
        assert out[1].isnan().all() and out[3].isnan().all()
    assert core.device_error() == 202
    keep = [0, 2]
    check_decode(q[keep], dict(c, table=c["table"][keep], lens=c["lens"][keep]), out[keep], inv_freq=inv_freq(D))
