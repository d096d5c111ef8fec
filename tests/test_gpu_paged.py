"""The paged key-value cache on the device against its definition in 64 bits (needs a B200).

Tolerances of `decode`.  Let u be the unit roundoff of the cache's type (half a step: bf16 2^-8,
f32 2^-24), A = |q| |k| * scale the size of a score's terms (an upper bound of their sum, by
Cauchy-Schwarz) and P = sum_j p_j |v_j|.

* scores, f32: D + 32 additions / products of relative error 2^-24 and cos / sin errors below
  2^-22 each side: |ds| <= (D + 64) 2^-24 A.
* scores, bf16: rotated keys and queries are exact fp32 values carried as hi + lo bf16 pieces;
  what the pieces drop is below 2^-16 each side plus the omitted lo.lo product, 2^-16:
  |ds| <= (3 * 2^-16 + (D + 64) 2^-24) A.
* p changes by at most a factor exp(2 |ds|) (numerator and normaliser), exp2 adds 2^-22; the
  probabilities enter P.V as hi + lo pieces (2^-16, bf16) and the sum of n terms adds n 2^-24.
* the result is rounded once: u |out|.
"""
import math

import pytest
import torch

import paged_ref as ref
from sta import core, paged
from sta.core import Geometry

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def on_gpu(c, weights=True):
    d = {n: x.cuda() for n, x in c.items()}
    return d, paged.PagedCache(d["k"], d["v"], d["table"], d["lens"], weights=d["weights"] if weights else None)


def queries(B, H, D, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((B, H, D), generator=g) * scale).to(dtype)


def inv_freq(D, theta=1e4):
    return 1.0 / (theta ** (torch.arange(0, D, 2, dtype=torch.float32) / D))


def relative_p(dtype, size, D, n):
    """Bound of an attention weight's relative error (see the module's docstring)."""
    ds = (3 * 2.0 ** -16 if dtype == torch.bfloat16 else 0.0) + (D + 64) * 2.0 ** -24
    return torch.expm1(2 * ds * size) + 2.0 ** -22 + (n + 64) * 2.0 ** -24


def check_decode(q, c, out, probs_out=None, **geo):
    D, dtype = q.shape[-1], q.dtype
    want, probs, mag, size = ref.decode(q, c, **geo)
    n = int(c["lens"].max()) if c["lens"].numel() else 0
    rel = relative_p(dtype, size, D, n)[..., None] + (2.0 ** -16 if dtype == torch.bfloat16 else 0.0)
    tol = U[dtype] * want.abs() + (1 + U[dtype]) * rel * mag + 1e-37
    err = (out.double().cpu() - want).abs()
    assert (err <= tol).all(), ((err / tol).max(), err.max())
    return probs, size


CASES = [
    # dtype, D, H, Hk, page, lens
    (torch.bfloat16, 128, 8, 2, 16, [1]),
    (torch.bfloat16, 128, 8, 2, 16, [0, 1, 15, 16, 17, 63, 64, 65, 200]),
    (torch.bfloat16, 128, 4, 4, 64, [129, 0, 640, 64]),
    (torch.bfloat16, 64, 4, 1, 1, [70, 5]),
    (torch.bfloat16, 64, 12, 2, 24, [333, 1000]),
    (torch.bfloat16, 128, 32, 2, 128, [700, 0, 0, 3]),
    (torch.bfloat16, 128, 3, 1, 100, [257]),
    (torch.bfloat16, 128, 2, 2, 256, [5000]),
    (torch.float32, 128, 8, 2, 16, [0, 1, 63, 64, 65, 300]),
    (torch.float32, 64, 4, 4, 8, [1, 1023, 0, 64]),
    (torch.float32, 64, 16, 1, 7, [450, 2]),
    (torch.float32, 128, 6, 2, 32, [1500]),
    (torch.float32, 64, 2, 1, 512, [2100, 40]),
]


@pytest.mark.parametrize("dtype,D,H,Hk,page,lens", CASES)
@pytest.mark.parametrize("geo", [dict(), dict(pos_scale=0.25, rope_scale=1.14), dict(dca=(192, 64), rope_scale=1.05)])
def test_decode(dtype, D, H, Hk, page, lens, geo):
    c = ref.make(lens, hk=Hk, D=D, page=page, dtype=dtype, seed=11, garbage=float("nan"))
    q = queries(len(lens), H, D, dtype, 12)
    d, cache = on_gpu(c)
    inv = inv_freq(D)
    g = Geometry(inv, geo.get("pos_scale", 1.0), geo.get("rope_scale", 1.0), geo.get("dca"))
    out = paged.decode(q.cuda(), cache, g)
    assert core.device_error() == 0
    check_decode(q, c, out, inv_freq=inv, **geo)
    # with the weights, once into a second array and once in place
    base = c["weights"].clone()
    w2 = torch.full_like(d["weights"], 7.0)
    out2 = paged.decode(q.cuda(), cache, g, weights_out=w2)
    out3 = paged.decode(q.cuda(), cache, g, weights_out=d["weights"])
    assert torch.equal(out2, out) and torch.equal(out3, out)
    _, probs, _, size = ref.decode(q, c, inv, **geo)
    want = ref.added_weights(c, probs, base)
    per_kv = relative_p(dtype, size, D, max(lens)).max().item()
    tol = 2.0 ** -24 * want + 1.01 * per_kv * (want - base.double()) + 1e-37
    live = torch.zeros(base.shape, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            live[c["table"][b, j // page], :, j % page] = True
    for got, rest in ((w2.cpu(), torch.full_like(base, 7.0)), (d["weights"].cpu(), base)):
        assert ((got.double() - want).abs() <= tol)[live].all()
        assert torch.equal(got[~live], rest[~live])  # slots without a key are left as they were


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_of_large_scores(dtype):
    """Peaked softmaxes: one key takes nearly all the weight."""
    lens, D = [900, 333], 128
    c = ref.make(lens, hk=2, D=D, page=16, dtype=dtype, seed=21, scale=4.0)
    q = queries(2, 8, D, dtype, 22, scale=4.0)
    _, cache = on_gpu(c)
    out = paged.decode(q.cuda(), cache, Geometry(inv_freq(D)))
    check_decode(q, c, out, inv_freq=inv_freq(D))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_at_far_positions(dtype):
    """Position 131071: angles up to 1.3e5 radians stay exact to fp32."""
    n, D = 131072, 64
    c = ref.make([n], hk=1, D=D, page=128, dtype=dtype, seed=23)
    q = queries(1, 2, D, dtype, 24, scale=2.0)
    _, cache = on_gpu(c)
    out = paged.decode(q.cuda(), cache, Geometry(inv_freq(D, 5e5)))
    check_decode(q, c, out, inv_freq=inv_freq(D, 5e5))


def test_decode_strides_and_wide_tables():
    """A pool laid out (pages, rows, heads, D), K and V interleaved, q a slice of a projection."""
    lens, D, Hk, H, page = [100, 37, 0], 128, 2, 8, 16
    c = ref.make(lens, hk=Hk, D=D, page=page, dtype=torch.bfloat16, seed=31, width=40)
    n_pages = c["k"].shape[0]
    pool = torch.empty((n_pages, page, 2, Hk, D), dtype=torch.bfloat16, device="cuda")
    k, v = pool[:, :, 0].transpose(1, 2), pool[:, :, 1].transpose(1, 2)
    k.copy_(c["k"])
    v.copy_(c["v"])
    wide = torch.full((3, 64), -1, dtype=torch.int32, device="cuda")
    wide[:, :40] = c["table"].cuda()
    cache = paged.PagedCache(k, v, wide[:, :50], c["lens"].cuda())
    q = queries(3, H, D, torch.bfloat16, 32)
    proj = torch.zeros((3, H + 5, D), dtype=torch.bfloat16, device="cuda")
    proj[:, 3:3 + H] = q.cuda()
    out = paged.decode(proj[:, 3:3 + H], cache, Geometry(inv_freq(D)))
    check_decode(q, c, out, inv_freq=inv_freq(D))


def test_decode_shares_pages_between_sequences():
    lens, D = [64, 64, 80], 64
    c = ref.make(lens, hk=1, D=D, page=16, dtype=torch.float32, seed=33)
    c["table"][1, :4] = c["table"][2, :4]  # a common prefix
    q = queries(3, 2, D, torch.float32, 34)
    _, cache = on_gpu(c)
    out = paged.decode(q.cuda(), cache, Geometry(inv_freq(D)))
    check_decode(q, c, out, inv_freq=inv_freq(D))


def test_pages_outside_the_pool():
    """A bad page makes its own sequence NaN, drops its rows and is reported; others are served."""
    lens, D, page = [40, 40, 40], 64, 16
    c = ref.make(lens, hk=2, D=D, page=page, dtype=torch.bfloat16, seed=35)
    n_pages = c["k"].shape[0]
    q = queries(3, 4, D, torch.bfloat16, 36)
    for bad in (-1, n_pages, 2 ** 31 - 1, -2 ** 31):
        cc = dict(c, table=c["table"].clone())
        cc["table"][1, 1] = bad
        d, cache = on_gpu(cc)
        w_out = torch.zeros_like(d["weights"])
        out = paged.decode(q.cuda(), cache, Geometry(inv_freq(D)), weights_out=w_out)
        assert core.device_error() == 202 and core.device_error() == 0
        assert out[1].isnan().all() and not out[0].isnan().any() and not out[2].isnan().any()
        keep = [0, 2]
        check_decode(q[keep], dict(c, table=c["table"][keep], lens=c["lens"][keep]), out[keep], inv_freq=inv_freq(D))
        new = torch.full((3, 2, 1, D), 5.0, dtype=torch.bfloat16, device="cuda")
        d["lens"].fill_(20)
        before = d["k"].clone()
        paged.append(cache, new, new)
        assert core.device_error() == 201
        assert torch.equal(d["lens"].cpu(), torch.tensor([21, 21, 21], dtype=torch.int32))
        changed = (d["k"] != before).flatten(1).any(1).nonzero().flatten().cpu().tolist()
        assert sorted(changed) == sorted([int(c["table"][0, 1]), int(c["table"][2, 1])])
        d["lens"].fill_(40)
        after, kept = paged.evict(cache, 8, c["free"][:3, None].cuda(), n_global=0, n_local=0)
        assert core.device_error() == 203
        want = ref.evict(c, 8, 0, 0)
        assert torch.equal(kept[keep].cpu(), want[keep]) and after.lens.tolist() == [8, 8, 8]
        paged.evict(cache, 32, torch.full((3, 2), bad, dtype=torch.int32, device="cuda"), n_global=0, n_local=0)
        assert core.device_error() == 203


def test_lengths_outside_the_table_are_clamped():
    lens, D = [32, 16], 64
    c = ref.make(lens, hk=1, D=D, page=16, dtype=torch.float32, seed=37)
    c["table"][1, 1] = c["free"][0]
    q = queries(2, 2, D, torch.float32, 38)
    d, cache = on_gpu(c)
    d["lens"].copy_(torch.tensor([1000, -5]))
    out = paged.decode(q.cuda(), cache, Geometry(inv_freq(D)))
    check_decode(q, dict(c, lens=torch.tensor([32, 0])), out, inv_freq=inv_freq(D))
    # rows past the table's last slot are dropped and reported
    d["lens"].copy_(torch.tensor([31, 30]))
    new = torch.ones((2, 1, 3, D), device="cuda")
    paged.append(cache, new, new)
    assert core.device_error() == 201
    assert d["lens"].tolist() == [32, 32]


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes: pages at its end are read, written and evicted."""
    D, page, n_pages = 128, 128, 140000  # 4.6 GB each for K and V
    k = torch.empty((n_pages, 1, page, D), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    w = torch.zeros((n_pages, 1, page), device="cuda")
    rows = torch.randn((1, 1, 300, D), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    last = torch.tensor([[n_pages - 1, n_pages - 3, 1]], dtype=torch.int32)
    cache = paged.PagedCache(k, v, last.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"), weights=w)
    paged.append(cache, rows.cuda(), rows.cuda() * 2)
    q = queries(1, 2, D, torch.bfloat16, 6)
    out = paged.decode(q.cuda(), cache, Geometry(inv_freq(D)), weights_out=w)
    small = dict(k=torch.zeros((3, 1, page, D), dtype=torch.bfloat16), lens=torch.tensor([300]),
                 table=torch.tensor([[0, 1, 2]], dtype=torch.int32))
    flat = torch.zeros((1, 1, 3 * page, D), dtype=torch.bfloat16)
    flat[:, :, :300] = rows
    small["k"] = flat.reshape(1, 1, 3, page, D).permute(2, 0, 1, 3, 4).reshape(3, 1, page, D)
    small["v"] = small["k"] * 2
    check_decode(q, small, out, inv_freq=inv_freq(D))
    after, kept = paged.evict(cache, 128, torch.tensor([[n_pages - 2]], dtype=torch.int32, device="cuda"))
    got = kept[0, 0].long()
    assert torch.equal(k[n_pages - 2, 0], rows[0, 0].cuda()[got])
    assert after.lens.item() == 128 and core.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,hk,page,lens,n,counts", [
    (128, 8, 16, [0, 1, 15, 16, 100], 1, None),
    (64, 3, 5, [0, 7, 23], 40, [40, 0, 13]),
    (128, 2, 24, [10, 0], 700, [700, 651]),
    (64, 1, 64, [5], 1, [0]),
    (128, 4, 128, [3, 9], 130, [-4, 1000]),  # clamped to 0 .. n
])
def test_append(dtype, D, hk, page, lens, n, counts):
    real = [n if counts is None else min(max(x, 0), n) for x in (counts or [n] * len(lens))]
    total = [a + b for a, b in zip(lens, real)]
    c = ref.make(total, hk=hk, D=D, page=page, dtype=dtype, seed=41)
    c["lens"] = torch.tensor(lens, dtype=torch.int32)
    g = torch.Generator().manual_seed(42)
    k_new = torch.randn((len(lens), n, hk, D), generator=g).to(dtype).transpose(1, 2)
    v_new = torch.randn((len(lens), n, hk, D), generator=g).to(dtype).transpose(1, 2)
    want = {x: c[x].clone() for x in ("k", "v", "weights")}
    for b in range(len(lens)):
        for i in range(real[b]):
            j = lens[b] + i
            pg, slot = int(c["table"][b, j // page]), j % page
            want["k"][pg, :, slot], want["v"][pg, :, slot] = k_new[b, :, i], v_new[b, :, i]
            want["weights"][pg, :, slot] = 0
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    unaligned = torch.zeros(len(lens) * n * hk * D + 1, dtype=dtype, device="cuda")[1:].view(len(lens), n, hk, D).transpose(1, 2)
    unaligned.copy_(k_new)
    for keys in (k_new.cuda(), k_new.cuda().contiguous(), unaligned):
        for in_place in (False, True):
            d, cache = on_gpu(c)
            out = None if in_place else torch.full((len(lens),), -9, dtype=torch.int32, device="cuda")
            got = paged.append(cache, keys, v_new.cuda(), counts=cnt, lens_out=out)
            assert core.device_error() == 0
            assert got.tolist() == total
            assert d["lens"].tolist() == (total if in_place else lens)
            for x in want:
                assert torch.equal(d[x].cpu(), want[x]), x


@pytest.mark.parametrize("n", [1, 90, 5000])  # one block per sequence, and many
def test_append_leaves_the_lengths_in_the_counts(n):
    lens, counts = [0, 10, 3], [n, n // 2, 0]
    total = [a + b for a, b in zip(lens, counts)]
    c = ref.make([n + 10] * 3, hk=4, D=64, page=16, dtype=torch.bfloat16, seed=44)
    c["lens"] = torch.tensor(lens, dtype=torch.int32)
    new = torch.randn((3, 4, n, 64), generator=torch.Generator().manual_seed(45)).bfloat16()
    want = c["k"].clone()
    for b in range(3):
        j = torch.arange(lens[b], total[b])
        want[c["table"][b, j // 16].long(), :, j % 16] = new[b, :, :counts[b]].transpose(0, 1)
    rows = new.cuda()
    for _ in range(5):
        d, cache = on_gpu(c)
        cnt = torch.tensor(counts, dtype=torch.int32, device="cuda")
        assert paged.append(cache, rows, rows, counts=cnt, lens_out=cnt) is cnt
        assert cnt.tolist() == total and d["lens"].tolist() == lens
        assert torch.equal(d["k"].cpu(), want)


def test_append_without_weights_and_of_nothing():
    c = ref.make([5], hk=2, D=64, page=4, dtype=torch.float32, seed=43)
    d, cache = on_gpu(c, weights=False)
    empty = torch.zeros((1, 2, 0, 64), device="cuda")
    assert paged.append(cache, empty, empty).tolist() == [5]
    assert torch.equal(d["k"].cpu(), c["k"])
    one = torch.ones((1, 2, 1, 64), device="cuda")
    paged.append(cache, one, one)
    assert d["lens"].tolist() == [6] and torch.equal(d["weights"].cpu(), c["weights"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,hk,page,lens,budget,n_global,n_local", [
    (128, 2, 16, [100, 64, 0, 1, 33], 32, 4, 4),
    (64, 1, 5, [257, 256, 255], 256, 0, 0),
    (128, 3, 24, [1000, 2500], 700, 32, 32),
    (64, 2, 64, [3000], 2999, 0, 1),
    (64, 2, 8, [50, 9], 8, 4, 4),       # nothing but forced keys
    (128, 1, 16, [40], 1, 0, 0),
    (64, 1, 256, [20, 10], 4096, 32, 32),  # budget above every length
    (64, 2, 128, [40000, 700], 3000, 4, 16),
])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_evict(dtype, D, hk, page, lens, budget, n_global, n_local, kind):
    c = ref.make(lens, hk=hk, D=D, page=page, dtype=dtype, seed=51, spare=3)
    g = torch.Generator().manual_seed(52)
    if kind == "ties":
        c["weights"] = torch.randint(0, 4, c["weights"].shape, generator=g).float()
    elif kind == "odd":
        u = torch.rand(c["weights"].shape, generator=g)
        w = torch.randn(c["weights"].shape, generator=g) * 10.0 ** torch.randint(-30, 30, u.shape, generator=g)
        for i, x in enumerate((0.0, -0.0, math.inf, -math.inf, math.nan, 1e-42)):
            w[(u > i * 0.05) & (u < (i + 1) * 0.05)] = x
        c["weights"] = w
    new = [min(n, budget) for n in lens]
    need = [-(-n // page) for n in new]
    n_pages = c["k"].shape[0]
    out_pages = torch.randperm(sum(need), generator=g).to(torch.int32) + n_pages
    for x in ("k", "v", "weights"):  # fresh pages behind the old ones
        c[x] = torch.cat((c[x], torch.full((sum(need) + 1,) + c[x].shape[1:], 9.0, dtype=c[x].dtype)))
    width = max(1, -(-min(budget, c["table"].shape[1] * page) // page))
    table_out = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table_out[b, :m] = out_pages[at:at + m]
        at += m
    want_kept = ref.evict(c, budget, n_global, n_local)
    d, cache = on_gpu(c)
    after, kept = paged.evict(cache, budget, table_out.cuda(), n_global=n_global, n_local=n_local)
    assert core.device_error() == 0
    assert after.lens.tolist() == new and d["lens"].tolist() == lens
    assert torch.equal(kept.cpu(), want_kept)
    for x in ("k", "v", "weights"):
        want = c[x].clone()
        for b, n in enumerate(new):
            r = torch.arange(n)
            for h in range(hk):
                src = want_kept[b, h, :n].long()
                pages = c["table"][b].long()[src // page]
                want[table_out[b].long()[r // page], h, r % page] = c[x][pages, h, src % page]
        got = d[x].cpu()
        assert torch.equal(torch.nan_to_num(got.float(), nan=-1.5), torch.nan_to_num(want.float(), nan=-1.5)), x


def test_evict_with_keys_in_a_workspace_of_odd_rows():
    """165005 slots a sequence (no multiple of four), two sequences of two heads, pages of five."""
    page, lens, budget = 5, [9001, 4003], 1999
    c = ref.make(lens, hk=2, D=64, page=page, dtype=torch.bfloat16, seed=53, spare=2 * 400, width=33001)
    d, cache = on_gpu(c)
    after, kept = paged.evict(cache, budget, c["free"][:800].reshape(2, 400).cuda(), n_global=3, n_local=5)
    assert core.device_error() == 0 and after.lens.tolist() == [budget] * 2
    assert torch.equal(kept.cpu(), ref.evict(c, budget, 3, 5))


def test_serving_run():
    """Prompts stored, steps decoded with their weights, the caches cut back, more steps: every
    step against the definition on what the cache holds then."""
    D, Hk, H, page, B = 64, 2, 8, 16, 3
    inv = inv_freq(D)
    geo = Geometry(inv.cuda(), 0.5, 1.1)
    g = torch.Generator().manual_seed(61)
    n_pages = 64
    k = torch.zeros((n_pages, Hk, page, D), dtype=torch.bfloat16, device="cuda")
    v, w = torch.zeros_like(k), torch.zeros((n_pages, Hk, page), device="cuda")
    pages = torch.randperm(n_pages, generator=g).to(torch.int32)
    table, spare = pages[:3 * 8].reshape(3, 8).cuda(), pages[24:24 + 3 * 4].reshape(3, 4)
    cache = paged.PagedCache(k, v, table, torch.zeros(B, dtype=torch.int32, device="cuda"), weights=w)
    prompt = [60, 1, 37]
    rows = torch.randn((2, B, Hk, max(prompt), D), generator=g).to(torch.bfloat16).cuda()
    paged.append(cache, rows[0], rows[1], counts=torch.tensor(prompt, dtype=torch.int32, device="cuda"))
    sums = torch.zeros((n_pages, Hk, page), dtype=torch.float64)
    for step in range(40):
        new = torch.randn((2, B, Hk, 1, D), generator=g).to(torch.bfloat16).cuda()
        paged.append(cache, new[0], new[1])
        q = torch.randn((B, H, D), generator=g).to(torch.bfloat16)
        now = dict(k=k.cpu(), v=v.cpu(), table=cache.table.cpu(), lens=cache.lens.cpu())
        out = paged.decode(q.cuda(), cache, geo, weights_out=w)
        probs, size = check_decode(q, now, out, inv_freq=inv, pos_scale=0.5, rope_scale=1.1)
        if step == 0:
            sums.zero_()
        sums = ref.added_weights(now, probs, sums)
        if step == 25:  # cut back into fresh pages (room for more steps), old pages given up
            assert (w.double().cpu() - sums).abs().max() <= relative_p(torch.bfloat16, size, D, 128).max() * 26 * 4
            wide = torch.cat((spare, pages[36:36 + 3 * 2].reshape(3, 2)), dim=1).cuda()
            was = dict(now, weights=w.cpu())
            cache, kept = paged.evict(cache, 48, wide, n_global=4, n_local=8)
            assert torch.equal(kept.cpu(), ref.evict(was, 48, 4, 8))
            assert cache.lens.tolist() == [48, 27, 48]
            sums = w.double().cpu()
    assert core.device_error() == 0


def test_graph_replay_and_streams():
    """A captured step (append, decode with weights, in place) replays on what the buffers hold
    then; two streams decode at once; results do not depend on either."""
    D, Hk, H, page, lens = 128, 2, 8, 16, [90, 200, 0]
    c = ref.make([n + 8 for n in lens], hk=Hk, D=D, page=page, dtype=torch.bfloat16, seed=71)
    c["lens"] = torch.tensor(lens, dtype=torch.int32)
    geo = Geometry(inv_freq(D).cuda())
    g = torch.Generator().manual_seed(72)
    steps = [(torch.randn((3, H, D), generator=g).to(torch.bfloat16).cuda(),
              torch.randn((3, Hk, 1, D), generator=g).to(torch.bfloat16).cuda()) for _ in range(4)]
    d, cache = on_gpu(c)
    want = []
    for q, x in steps:
        paged.append(cache, x, x)
        want.append((paged.decode(q, cache, geo, weights_out=d["weights"]), d["weights"].clone()))
    torch.cuda.synchronize()
    d, cache = on_gpu(c)
    q_buf, x_buf = steps[0][0].clone(), steps[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            paged.append(cache, x_buf, x_buf)
            out = paged.decode(q_buf, cache, geo, weights_out=d["weights"])
    for (q, x), (o, w) in zip(steps, want):
        q_buf.copy_(q)
        x_buf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(d["weights"], w)
    # two calls at once on streams of their own
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    first = [paged.decode(steps[i][0], cache, geo) for i in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged.decode(steps[i][0], cache, geo))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, first[i]) for o in outs[i])


def test_python_refusals():
    c = ref.make([5, 6], hk=2, D=64, page=4, dtype=torch.float32, seed=81)
    d, cache = on_gpu(c)
    geo = Geometry(inv_freq(64))
    q = torch.zeros((2, 4, 64), device="cuda")
    with pytest.raises(TypeError):
        paged.decode(q.bfloat16(), cache, geo)
    with pytest.raises(ValueError):
        paged.decode(q[:1], cache, geo)
    with pytest.raises(ValueError):
        paged.decode(q[:, :3], cache, geo)
    with pytest.raises(ValueError):
        paged.decode(q.cpu(), cache, geo)
    with pytest.raises(ValueError):
        paged.decode(q, cache, Geometry(inv_freq(128)))
    with pytest.raises(ValueError):
        paged.decode(q, cache, Geometry(inv_freq(64), 1.0, 1.0, (100, 60)))
    with pytest.raises(ValueError):
        paged.decode(q, cache, geo, weights_out=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError):
        paged.decode(q, paged.PagedCache(d["k"], d["v"], d["table"], d["lens"]), geo, weights_out=d["weights"])
    with pytest.raises(TypeError):
        paged.PagedCache(d["k"].half(), d["v"].half(), d["table"], d["lens"])
    with pytest.raises(TypeError):
        paged.PagedCache(d["k"], d["v"], d["table"].long(), d["lens"])
    with pytest.raises(ValueError):
        paged.PagedCache(d["k"], d["v"][:1], d["table"], d["lens"])
    with pytest.raises(ValueError):
        paged.PagedCache(d["k"].transpose(2, 3), d["v"], d["table"], d["lens"])
    with pytest.raises(ValueError):
        paged.evict(cache, 4, d["table"], n_global=3, n_local=3)
    with pytest.raises(ValueError):
        paged.evict(cache, 6, d["table"][:, :1], n_global=0, n_local=0)
    with pytest.raises(ValueError):
        paged.append(cache, q, q)
    with pytest.raises(TypeError):
        paged.append(cache, q[:, :2, None], q[:, :2, None], counts=torch.zeros(2, device="cuda"))


def test_outputs_do_not_depend_on_the_other_sequences():
    """Deterministic, and the same bits twice."""
    lens, D = [3000, 10, 777], 128
    c = ref.make(lens, hk=2, D=D, page=16, dtype=torch.bfloat16, seed=91)
    _, cache = on_gpu(c)
    q = queries(3, 8, D, torch.bfloat16, 92).cuda()
    a = paged.decode(q, cache, Geometry(inv_freq(D)))
    b = paged.decode(q, cache, Geometry(inv_freq(D)))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,D,G", [(torch.bfloat16, 64, 20), (torch.bfloat16, 128, 33), (torch.bfloat16, 128, 12),
                                       (torch.float32, 128, 8), (torch.float32, 64, 19)])
def test_decode_of_many_heads_per_kv_head(dtype, D, G):
    """Groups of q heads that one pass over the keys cannot serve."""
    lens = [333, 64, 0, 17]
    c = ref.make(lens, hk=2, D=D, page=32, dtype=dtype, seed=101)
    q = queries(4, 2 * G, D, dtype, 102)
    d, cache = on_gpu(c)
    w = torch.zeros_like(d["weights"])
    out = paged.decode(q.cuda(), cache, Geometry(inv_freq(D)), weights_out=w)
    probs, size = check_decode(q, c, out, inv_freq=inv_freq(D))
    want = ref.added_weights(c, probs, c["weights"])
    rel = relative_p(dtype, size, D, 333).max().item()
    got = torch.where(w.cpu() == 0, want, w.cpu().double())  # slots without a key stay zero
    assert ((got - want).abs() <= 2.0 ** -24 * want + 1.01 * rel * (want - c["weights"].double())).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,lens", [
    (16, [int(7.7 * i) % 90 if i % 5 else 0 for i in range(77)]),      # more sequences than lanes
    (24, [0] * 40 + [700] + [0] * 30 + [3, 0]),
    (64, [0] * 35),
    (256, [33]),
])
def test_decode_of_many_and_empty_sequences(dtype, page, lens):
    c = ref.make(lens, hk=2, D=64, page=page, dtype=dtype, seed=103)
    q = queries(len(lens), 4, 64, dtype, 104)
    _, cache = on_gpu(c)
    out = paged.decode(q.cuda(), cache, Geometry(inv_freq(64)))
    check_decode(q, c, out, inv_freq=inv_freq(64))


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float32, 128), (torch.float32, 64)])
@pytest.mark.parametrize("page", [8, 16, 24, 100])
def test_a_bad_page_reaches_its_own_sequence_only(dtype, D, page):
    lens = [300, 290, 310]
    c = ref.make(lens, hk=2, D=D, page=page, dtype=dtype, seed=105)
    c["table"][1, 2] = c["k"].shape[0] + 5
    q = queries(3, 8, D, dtype, 106)
    _, cache = on_gpu(c)
    out = paged.decode(q.cuda(), cache, Geometry(inv_freq(D)))
    assert core.device_error() == 202
    assert out[1].isnan().all()
    keep = [0, 2]
    check_decode(q[keep], dict(c, table=c["table"][keep], lens=c["lens"][keep]), out[keep], inv_freq=inv_freq(D))


def test_evict_of_more_slots_than_shared_memory_holds():
    """A table that names 204800 slots: the selection keeps its keys in the workspace."""
    page, lens, budget = 4096, [150001, 300], 70000
    c = ref.make(lens, hk=1, D=64, page=page, dtype=torch.bfloat16, seed=107, width=50, spare=20)
    g = torch.Generator().manual_seed(108)
    c["weights"] = torch.randint(0, 5000, c["weights"].shape, generator=g).float()
    table_out = torch.full((2, 18), -1, dtype=torch.int32)
    table_out[0] = c["free"][:18]
    table_out[1, 0] = c["free"][18]
    d, cache = on_gpu(c)
    after, kept = paged.evict(cache, budget, table_out.cuda(), n_global=4, n_local=8)
    assert core.device_error() == 0 and after.lens.tolist() == [70000, 300]
    want = ref.evict(c, budget, 4, 8)
    assert torch.equal(kept.cpu(), want)
    j = want[0, 0].long()
    src = c["k"][c["table"][0].long()[j // page], 0, j % page]
    r = torch.arange(budget)
    assert torch.equal(d["k"].cpu()[table_out[0].long()[r // page], 0, r % page], src)


def test_evict_in_a_graph():
    lens, D, page = [400, 90], 64, 16
    c = ref.make(lens, hk=2, D=D, page=page, dtype=torch.float32, seed=109, spare=20)
    table_out = c["free"][:16].reshape(2, 8)
    d, cache = on_gpu(c)
    out_dev = table_out.cuda()
    paged.evict(cache, 128, out_dev, n_global=2, n_local=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            after, kept = paged.evict(cache, 128, out_dev, n_global=2, n_local=2)
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        c["weights"] = torch.rand(c["weights"].shape, generator=g)
        d["weights"].copy_(c["weights"])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept.cpu(), ref.evict(c, 128, 2, 2)) and after.lens.tolist() == [128, 90]


def test_an_empty_batch():
    c = ref.make([5], hk=2, D=64, page=4, dtype=torch.float32, seed=110)
    d, _ = on_gpu(c)
    cache = paged.PagedCache(d["k"], d["v"], d["table"][:0], d["lens"][:0], weights=d["weights"])
    assert paged.decode(torch.zeros((0, 4, 64), device="cuda"), cache, Geometry(inv_freq(64))).shape == (0, 4, 64)
    assert paged.append(cache, torch.zeros((0, 2, 1, 64), device="cuda"), torch.zeros((0, 2, 1, 64), device="cuda")).numel() == 0
    after, kept = paged.evict(cache, 4, torch.zeros((0, 1), dtype=torch.int32, device="cuda"), n_global=0, n_local=0)
    assert kept.shape == (0, 2, 4) and after.lens.numel() == 0


def test_more_sequences_than_a_grid_dimension():
    B, D = 66000, 64
    k = torch.zeros((B, 1, 2, D), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.arange(B, dtype=torch.int32, device="cuda").flip(0)[:, None].contiguous()
    lens = (torch.arange(B, device="cuda") % 2).to(torch.int32)
    cache = paged.PagedCache(k, v, table, lens)
    rows = torch.randn((B, 1, 1, D), device="cuda").to(torch.bfloat16)
    paged.append(cache, rows, rows)
    at = torch.arange(B, device="cuda")
    assert torch.equal(k[table[:, 0].long(), 0, at % 2], rows[:, 0, 0])
    assert torch.equal(lens, (at % 2 + 1).to(torch.int32))
    out = paged.decode(rows[:, 0].expand(B, 2, D), cache, Geometry(inv_freq(D)))
    one = at % 2 == 0  # a single key: the output is its value
    assert torch.equal(out[one, 0], rows[one, 0, 0])
    with pytest.raises(ValueError):
        paged.evict(paged.PagedCache(k, v, table, lens, weights=torch.zeros((B, 1, 2), device="cuda")), 1, table,
                    n_global=0, n_local=0)


def test_steps_in_a_row_do_not_overtake_each_other():
    """Appends and decodes with weights in place, back to back without a wait: each kernel sees what
    the ones ahead of it wrote."""
    D, Hk, H, page, B = 64, 2, 4, 16, 4
    pages = torch.arange(B * 20, dtype=torch.int32).reshape(B, 20)
    g = torch.Generator().manual_seed(111)
    xs = torch.randn((60, B, Hk, 1, D), generator=g).to(torch.bfloat16).cuda()
    qs = torch.randn((60, B, H, D), generator=g).to(torch.bfloat16).cuda()
    geo = Geometry(inv_freq(D).cuda())
    results = []
    for wait in (True, False):
        k = torch.zeros((B * 20, Hk, page, D), dtype=torch.bfloat16, device="cuda")
        v, w = torch.zeros_like(k), torch.ones((B * 20, Hk, page), device="cuda")
        cache = paged.PagedCache(k, v, pages.cuda(), torch.tensor([0, 100, 200, 7], dtype=torch.int32, device="cuda"), weights=w)
        outs = []
        torch.cuda.synchronize()
        for x, q in zip(xs, qs):
            paged.append(cache, x, x)
            if wait:
                torch.cuda.synchronize()
            outs.append(paged.decode(q, cache, geo, weights_out=w))
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        results.append((torch.stack(outs), w, cache.lens))
    for a, b in zip(*results):
        assert torch.equal(a, b)
