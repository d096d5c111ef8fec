"""The paged key-value cache: calls that the documentation allows and the first set of tests does
not make (needs a B200)."""
import math

import pytest
import torch

import paged_ref as ref
from sta import core, paged
from sta.core import Geometry
from test_gpu_paged import check_decode, inv_freq, on_gpu, queries, relative_p

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


def test_a_bad_page_is_not_taken_for_an_expired_wait():
    """The prefill hooks ask for expired waits after every layer; what a paged cache has reported by
    then is not one, and is still there for who asks."""
    from sta import hooks
    c = ref.make([5], hk=1, D=64, page=4, dtype=torch.float32, seed=203)
    c["table"][0, 1] = -1
    _, cache = on_gpu(c)
    assert core.device_error() == 0
    paged.decode(torch.ones((1, 1, 64), device="cuda"), cache, Geometry(inv_freq(64).cuda()))
    hooks._check_device_waits()
    assert core.wait_error() == 0
    assert core.device_error() == 202
    assert core.device_error() == 0


def test_an_expired_wait_and_a_bad_page_are_both_reported():
    q = torch.randn((8, 4096, 128), generator=torch.Generator().manual_seed(204)).bfloat16().cuda()
    c = ref.make([5], hk=1, D=64, page=4, dtype=torch.float32, seed=203)
    c["table"][0, 1] = -1
    _, cache = on_gpu(c)
    assert core.device_error() == 0
    paged.decode(torch.ones((1, 1, 64), device="cuda"), cache, Geometry(inv_freq(64).cuda()))
    core.select(q, q[:2], torch.full((8,), 5.0), Geometry(inv_freq(128)), tile=64, wait_limit_ns=1)
    assert core.device_error() in (101, 102, 103, 104)
    assert core.device_error() == 202
    assert core.device_error() == 0


def test_a_capture_survives_the_refusal_of_frequencies_elsewhere():
    c = ref.make([40], hk=2, D=64, page=16, dtype=torch.bfloat16, seed=205)
    _, cache = on_gpu(c)
    q = queries(1, 4, 64, torch.bfloat16, 206).cuda()
    there = Geometry(inv_freq(64).cuda())
    want = paged.decode(q, cache, Geometry(inv_freq(64)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(ValueError):
                paged.decode(q, cache, Geometry(inv_freq(64)))
            out = paged.decode(q, cache, there)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def weights_of(c, probs, base, b):
    """What sequence b alone makes of the weights."""
    return ref.added_weights(c, [p if i == b else p[:, :0] for i, p in enumerate(probs)], base)


@pytest.mark.parametrize("dtype,D,page", [(torch.bfloat16, 128, 16), (torch.bfloat16, 64, 6), (torch.float32, 64, 16)])
def test_weights_of_a_page_that_stands_in_the_table_twice(dtype, D, page):
    """One of its places adds to them, the others are dropped and reported; pages of one sequence
    alone are as ever.  Entries that are not in use may name any page."""
    lens, hk, H = [64, 64, 80, 33], 2, 4
    c = ref.make(lens, hk=hk, D=D, page=page, dtype=dtype, seed=207, width=20)
    q = queries(4, H, D, dtype, 208)
    geo = Geometry(inv_freq(D).cuda())
    own = dict(c, table=c["table"].clone())
    c["table"][3, -(-33 // page):] = c["table"][0, 0]  # not in use
    d, cache = on_gpu(c)
    out = paged.decode(q.cuda(), cache, geo, weights_out=d["weights"])
    assert core.device_error() == 0
    check_decode(q, c, out, inv_freq=inv_freq(D))
    c["table"][1, :2] = c["table"][2, :2]  # a common prefix
    c["table"][0, 3] = c["table"][0, 1]    # and one page twice in a sequence
    d, cache = on_gpu(c)
    for in_place in (False, True):
        base = d["weights"].cpu()
        got = d["weights"] if in_place else torch.full_like(d["weights"], -1.0)
        out = paged.decode(q.cuda(), cache, geo, weights_out=got)
        assert core.device_error() == 204 and core.device_error() == 0
        check_decode(q, c, out, inv_freq=inv_freq(D))
        got = got.cpu().double()
        _, probs, _, size = ref.decode(q, c, inv_freq(D))
        alone = [weights_of(c, probs, base, b) for b in range(4)]
        # a key's added weight is below H / hk = 2, its sum below 4 (rounded to 2^-23); a lost or doubled
        # update is off by about 1 / 32 on a page
        tol = 2 * relative_p(dtype, size, D, 80).max() + 2.0 ** -22
        assert tol < 1 / 64
        for t in range(2):
            pg = int(c["table"][2, t])
            assert min((got[pg] - alone[b][pg]).abs().max() for b in (1, 2)) < tol
        for b, t in ((1, 3), (2, 2), (3, 0), (0, 0)):
            pg = int(c["table"][b, t])
            assert (got[pg] - alone[b][pg])[:, :min(page, lens[b] - t * page)].abs().max() < tol
        pg, n = int(c["table"][0, 1]), probs[0].shape[1]
        p = probs[0].reshape(hk, H // hk, n).sum(1)
        first, again = (base[pg].double() + p[:, t * page:(t + 1) * page] for t in (1, 3))
        assert min((got[pg] - x).abs().max() for x in (first, again)) < tol


@pytest.mark.parametrize("dtype,page,lens,budget", [
    (torch.bfloat16, 16, [300, 200, 40, 33], 48),
    (torch.float32, 5, [300, 90, 48, 7], 48),
    (torch.bfloat16, 64, [20000, 9000, 100, 48], 1000),   # clusters, several entries per thread and none
    (torch.float32, 1, [50, 3000, 48, 9], 48),
])
@pytest.mark.parametrize("kind", ["in use", "in use by a sequence that is kept whole", "twice", "twice in a sequence"])
def test_evict_into_pages_that_are_not_free(dtype, page, lens, budget, kind):
    """Rows of the cache are never overwritten; of a new page named twice one entry's rows are
    written; the other new pages are as ever, and the call is reported."""
    hk, D = 2, 64
    new = [min(n, budget) for n in lens]
    need = [-(-n // page) for n in new]
    c = ref.make(lens, hk=hk, D=D, page=page, dtype=dtype, seed=209, spare=sum(need) + 2)
    table_out = torch.full((4, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table_out[b, :m] = c["free"][at:at + m]
        at += m
    free = int(c["free"][at])
    want_kept = ref.evict(c, budget, 2, 2)
    d, cache = on_gpu(c)
    before = {x: d[x].clone() for x in ("k", "v", "weights")}
    entries = {"in use": [(0, 0)], "in use by a sequence that is kept whole": [(1, 0)], "twice": [(0, 0), (1, 0)],
               "twice in a sequence": [(0, 0), (0, need[0] - 1)]}[kind]
    odd = free if kind.startswith("twice") else int(c["table"][0 if kind == "in use" else 3, 0])
    used = {int(x) for b, n in enumerate(lens) for x in c["table"][b, :-(-n // page)]}
    assert (odd in used) != kind.startswith("twice")
    for b, t in entries:
        table_out[b, t] = odd
    c["table"][3, need[3]:] = table_out[2, 0]  # not in use
    d["table"].copy_(c["table"])
    for _ in range(3):
        for x in before:
            d[x].copy_(before[x])
        after, kept = paged.evict(cache, budget, table_out.cuda(), n_global=2, n_local=2)
        assert core.device_error() == 204 and core.device_error() == 0
        assert torch.equal(kept.cpu(), want_kept) and after.lens.tolist() == new

        def rows(b, t, x):  # what entry t of sequence b brings: (heads, rows, ...)
            r = want_kept[b, :, t * page:min(new[b], (t + 1) * page)].long()
            return torch.stack([c[x][c["table"][b].long()[r[h] // page], h, r[h] % page] for h in range(hk)])

        for x in before:
            got = d[x].cpu()
            want = before[x].cpu()
            for b in range(4):
                for t in range(need[b]):
                    pg = int(table_out[b, t])
                    y = rows(b, t, x)
                    if pg != odd:
                        want[pg, :, :y.shape[1]] = y
            if odd not in used:  # one entry's rows
                ys = [rows(b, t, x) for b, t in entries]
                left = [torch.equal(got[odd, :, :y.shape[1]], y) for y in ys]
                assert any(left)
                got[odd] = want[odd]
            assert torch.equal(got, want), x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,wide,first", [(16, 17, 0), (8, 9, 0), (64, 64, 1), (4, 6, 2)])
def test_weights_that_cannot_be_read_four_at_a_time(dtype, page, wide, first):
    """Pages of a multiple of four whose weights have other strides, or begin between boundaries."""
    lens, D, hk, H = [300, 17, 0, 65], 64, 2, 4
    c = ref.make(lens, hk=hk, D=D, page=page, dtype=dtype, seed=211, spare=40)
    n_pages = c["k"].shape[0]
    d, _ = on_gpu(c)
    flat = torch.full((n_pages * hk * wide + 4,), -3.0, device="cuda")
    w, w2 = (flat.clone().as_strided((n_pages, hk, page), (hk * wide, wide, 1), first) for _ in range(2))
    w.copy_(d["weights"])
    cache = paged.PagedCache(d["k"], d["v"], d["table"], d["lens"], weights=w)
    q = queries(4, H, D, dtype, 212)
    geo = Geometry(inv_freq(D).cuda())
    out = paged.decode(q.cuda(), cache, geo, weights_out=w2)
    assert core.device_error() == 0
    probs, size = check_decode(q, c, out, inv_freq=inv_freq(D))
    want = ref.added_weights(c, probs, c["weights"])
    live = torch.zeros(w.shape, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            live[c["table"][b, j // page], :, j % page] = True
    tol = 2.0 ** -24 * want + 1.01 * relative_p(dtype, size, D, 300).max() * (want - c["weights"].double())
    assert ((w2.cpu().double() - want).abs() <= tol)[live].all()
    assert (w2.cpu()[~live] == -3).all()
    # and the selection reads them
    need = -(-32 // page)
    table_out = c["free"][:4 * need].reshape(4, need) if 4 * need <= len(c["free"]) else None
    assert table_out is not None
    after, kept = paged.evict(cache, 32, table_out.cuda(), n_global=2, n_local=2)
    assert core.device_error() == 0
    assert torch.equal(kept.cpu(), ref.evict(c, 32, 2, 2))
    held = torch.full(flat.shape, True)
    for pg in range(n_pages):
        for h in range(hk):
            held[first + (pg * hk + h) * wide:first + (pg * hk + h) * wide + page] = False
    base = w._base if w._base is not None else w
    assert (base.flatten().cpu()[held] == -3).all()  # nothing between the rows is written


@pytest.mark.parametrize("dtype,page,prefix", [(torch.bfloat16, 16, 6), (torch.float32, 5, 20)])
def test_a_shared_prefix_until_every_sequence_has_pages_of_its_own(dtype, page, prefix):
    """Sequences that share their first pages are decoded without weights, cut into fresh pages (old
    pages may be shared), and go on with weights: a narrow slice of a wide table serves them."""
    D, hk, H, n = 64, 2, 4, prefix * page
    lens = [n + 30, n + 3, n + 57]
    c = ref.make(lens, hk=hk, D=D, page=page, dtype=dtype, seed=213, spare=120, width=100)
    for b in (1, 2):
        c["table"][b, :prefix] = c["table"][0, :prefix]
    d, _ = on_gpu(c)
    geo = Geometry(inv_freq(D).cuda())
    whole = paged.PagedCache(d["k"], d["v"], d["table"], d["lens"], weights=d["weights"])
    cache = whole.with_pages(d["table"][:, :-(-max(lens) // page)], d["lens"])
    q = queries(3, H, D, dtype, 214)
    out = paged.decode(q.cuda(), cache, geo)
    assert torch.equal(paged.decode(q.cuda(), whole, geo), out)
    check_decode(q, c, out, inv_freq=inv_freq(D))
    budget = n + 10
    need = -(-(budget + 8) // page)
    table_out = c["free"][:3 * need].reshape(3, need)
    after, kept = paged.evict(cache, budget, table_out.cuda(), n_global=4, n_local=4)
    want = ref.evict(c, budget, 4, 4)
    assert core.device_error() == 0 and torch.equal(kept.cpu(), want)
    assert after.lens.tolist() == [budget, n + 3, budget]
    for b, m in enumerate((budget, n + 3, budget)):
        r = torch.arange(m)
        for h in range(hk):
            src = want[b, h, :m].long()
            for x in ("k", "v", "weights"):
                got = d[x].cpu()[table_out[b].long()[r // page], h, r % page]
                assert torch.equal(got, c[x][c["table"][b].long()[src // page], h, src % page])
    for step in range(8):  # room for them in the fresh pages
        new = torch.randn((2, 3, hk, 1, D), generator=torch.Generator().manual_seed(step)).to(dtype).cuda()
        paged.append(after, new[0], new[1])
        now = dict(k=d["k"].cpu(), v=d["v"].cpu(), table=table_out, lens=after.lens.cpu())
        base = d["weights"].cpu()
        out = paged.decode(q.cuda(), after, geo, weights_out=d["weights"])
        probs, size = check_decode(q, now, out, inv_freq=inv_freq(D))
        want = ref.added_weights(now, probs, base)
        rel = relative_p(dtype, size, D, max(lens)).max()
        assert ((d["weights"].cpu().double() - want).abs() <= 2.0 ** -24 * want + 1.01 * rel * (want - base.double())).all()
    assert core.device_error() == 0
