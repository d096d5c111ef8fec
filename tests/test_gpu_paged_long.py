"""Decode over paged caches that are long enough for the kernels' steady state: shares of many units
(bf16: more than 32 tiles, so that the running angle is renewed inside a share), rings that are
refilled, joins inside a CTA (needs a B200).

The data make every unit of 16 keys count.  A value has one dim that is not zero, that of its unit
(unit number modulo D), with the unit's sign and a magnitude in 1 .. 2: a dim of the result sums the
n / 16 / D units of one residue, so a unit that is dropped or taken twice moves it by D * 16 / n of
the sum of p |v|.  Queries are short (scores of standard deviation 0.4), so all keys have weights of
one order; the weights are compared key by key, each relative to itself, which no wrong rotation,
page or order survives (a shift by 0.05 positions moves most weights by some 1 %).

Tolerances.  u is half a step of the output's type (bf16 2^-8, f32 2^-24), A = |q| |k| * scale.
* a rotated key enters the products as hi + lo bf16 pieces: cutting hi leaves less than 2^-7 of the
  value, rounding that to lo 2^-8 of the rest, 2^-15; queries are rounded twice, 2^-16; all four
  products are formed.  With the fp32 rotation (running products of at most 32 turns, 2^-24 each, and
  a few roundings) and the sum over D: |ds| <= (3 * 2^-16 + (D + 64) 2^-24) A; f32 the latter alone.
* p moves by exp(2 |ds|) at most (numerator and sum) and 2^-22 of exp2; in P.V p is hi + lo, 2^-16.
* sums: a share adds its units one after the other (bf16: two products of 16 keys, each of which may
  lose 2^-22 of the sum; f32: its eight keys of a tile in a warp, counted alike), a CTA joins its shares, and
  a warp of the join adds every fourth or sixteenth of at most W partials: depth * 2^-22 in all.
* the result is rounded once.
"""
import math

import pytest
import torch

from sta import core, paged
from sta.core import Geometry
from test_gpu_paged import inv_freq

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMS = 148
PI, FAR, NEAR = dict(pos_scale=0.25, rope_scale=1.14), dict(dca=(6144, 1024)), dict(dca=(192, 64), rope_scale=1.05)


def shares(dtype, D, G, lens, hk):
    """Shares at most, units of a share (rounded up), and q heads of one pass, as the kernels cut them."""
    if dtype is torch.float32:
        gt, unit, w = (8 if G > 4 else 4 if G > 2 else G), 64, (1 if D == 128 else 2) * SMS
    else:
        gt, unit = (16 if G > 8 else 8), 16
        w = {(128, 8): 12, (128, 16): 8, (64, 8): 16, (64, 16): 12}[D, gt] * SMS
    total = sum(-(-n // unit) for n in lens) * hk * -(-G // gt)
    return w, -(-total // w), gt


def make(lens, hk, D, page, dtype, seed, layout):
    """Pools, tables and weights on the device; layout: 'dense' or 'rows' (K and V interleaved, heads inside rows)."""
    g = torch.Generator("cuda").manual_seed(seed)
    used = [-(-n // page) for n in lens]
    n_pages = sum(used) + 2
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(used)), -1, dtype=torch.int32, device="cuda")
    if layout == "rows":
        pool = torch.empty((n_pages, page, 2, hk, D), dtype=dtype, device="cuda")
        k, v = pool[:, :, 0].transpose(1, 2), pool[:, :, 1].transpose(1, 2)
    else:
        k, v = (torch.empty((n_pages, hk, page, D), dtype=dtype, device="cuda") for _ in range(2))
    for part in k.split(2048):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    v.fill_(float("nan"))
    at = 0
    for b, m in enumerate(used):
        table[b, :m] = order[at:at + m]
        at += m
        j = torch.arange(m * page, device="cuda")
        sign = (torch.randint(0, 2, (m * page // 16 + 1,), generator=g, device="cuda") * 2 - 1)[j // 16]
        n = lens[b]
        if m > 0:  # what lies behind the last token is never read
            k[table[b, m - 1].long(), :, n - (m - 1) * page:] = float("nan")
        x = (1 + torch.rand((hk, m * page), generator=g, device="cuda")) * sign
        rows = torch.zeros((hk, m * page, D), device="cuda")
        rows.scatter_(2, (j // 16 % D).expand(hk, -1)[..., None], x[..., None])
        rows[:, n:] = float("nan")
        v[table[b, :m].long()] = rows.reshape(hk, m, page, D).transpose(0, 1).to(dtype)
    w = torch.rand((n_pages, hk, page), generator=g, device="cuda")
    return dict(k=k, v=v, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), weights=w)


def rows_of(c, b, n, name):
    page = c["k"].shape[2]
    m = -(-n // page)
    x = c[name][c["table"][b, :m].long()].transpose(0, 1)
    return x.reshape((x.shape[0], m * page) + x.shape[3:])[:, :n]


def rotated(x, pos, inv, scale):
    a = pos[:, None] * inv
    co, si = a.cos() * scale, a.sin() * scale
    x1, x2 = x.chunk(2, -1)
    return torch.cat((x1 * co - x2 * si, x2 * co + x1 * si), -1)


def definition(q, c, b, inv, pos_scale=1.0, rope_scale=1.0, dca=None):
    """Sequence b in 64 bits: out (H, D), weights (hk, G, n), sum of p |v| (H, D), largest A per head (H, 1)."""
    n, hk, D = int(c["lens"][b]), c["k"].shape[1], q.shape[-1]
    inv, sm = inv.double(), 1.0 / math.sqrt(D)
    j, i = torch.arange(n, device="cuda"), n - 1
    if dca is None:
        key_pos, query_pos, which = j.double() * pos_scale, [i * pos_scale], torch.zeros_like(j)
    else:
        s, w = dca
        L = s - w
        key_pos, which = (j % L).double(), (i // L - j // L).clamp(max=2)
        query_pos = [i % L, min(L + i % L, s), min(2 * L - 1, s)]
    at = torch.tensor(query_pos, dtype=torch.float64, device="cuda")
    outs, mags, sizes, probs = [], [], [], []
    qs = q[b].double().reshape(hk, -1, D)
    k, v = rows_of(c, b, n, "k"), rows_of(c, b, n, "v")
    for h in range(hk):
        kr = rotated(k[h].double(), key_pos, inv, rope_scale)
        x = torch.stack([rotated(qs[h], at[m].expand(qs.shape[1]), inv, rope_scale) @ kr.t() for m in range(len(at))])
        p = torch.softmax(x.gather(0, which.expand(1, qs.shape[1], n))[0] * sm, dim=-1)
        outs.append(p @ v[h].double())
        mags.append(p @ v[h].double().abs())
        sizes.append(qs[h].norm(dim=-1, keepdim=True) * k[h].double().norm(dim=-1).max() * rope_scale ** 2 * sm)
        probs.append(p)
    return torch.cat(outs), torch.stack(probs), torch.cat(mags), torch.cat(sizes)


def run(dtype, D, G, hk, page, lens, geo, layout="dense", seed=0, q=None, tiles=1):
    """A decode with and without weights against the definition."""
    c = make(lens, hk, D, page, dtype, seed, layout)
    w_most, per_share, _ = shares(dtype, D, G, lens, hk)
    assert per_share >= tiles * (4 if dtype is torch.bfloat16 else 1)
    H = hk * G
    if q is None:
        g = torch.Generator("cuda").manual_seed(seed + 1)
        q = (torch.randn((len(lens), H, D), generator=g, device="cuda") * 0.4).to(dtype)
    inv = inv_freq(D).cuda()
    cache = paged.PagedCache(c["k"], c["v"], c["table"], c["lens"], weights=c["weights"])
    g = Geometry(inv, geo.get("pos_scale", 1.0), geo.get("rope_scale", 1.0), geo.get("dca"))
    got_w = torch.zeros_like(c["weights"])
    out = paged.decode(q, cache, g, weights_out=got_w)
    assert core.device_error() == 0
    assert torch.equal(paged.decode(q, cache, g), out)
    depth = (2 if dtype is torch.bfloat16 else 8) * per_share + w_most / 4 + 64
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].any()
            continue
        want, p, mag, size = definition(q, c, b, inv, **geo)
        ds = (3 * 2.0 ** -16 if dtype is torch.bfloat16 else 0.0) + (D + 64) * 2.0 ** -24
        rel = torch.expm1(2 * ds * size) + depth * 2.0 ** -22
        assert rel.max() < 0.01  # sharp enough for what the data show
        tol = U[dtype] * want.abs() + (1 + U[dtype]) * (rel + 2.0 ** -16) * mag
        err = (out[b].double() - want).abs()
        assert (err <= tol).all(), (b, (err / tol).max())
        base = rows_of(c, b, n, "weights").double()
        add = p.sum(1)
        err = (rows_of(dict(c, w=got_w), b, n, "w").double() - (base + add)).abs()
        tol = 2.0 ** -23 * (base + add) + rel.max() * 1.01 * add
        assert (err <= tol).all(), (b, (err / tol).max())


# sums to 465 k keys: 131 units a share of 1776, shares begin and end inside tiles
LENS = [131067, 100003, 77777, 65536, 50001, 41009, 0, 13]


@pytest.mark.parametrize("D,G,page,layout,geo", [
    (128, 4, 16, "dense", {}), (128, 4, 24, "dense", PI), (128, 4, 64, "rows", FAR), (128, 4, 128, "dense", NEAR),
    (128, 12, 16, "dense", NEAR), (128, 12, 24, "dense", {}), (128, 12, 64, "rows", PI), (128, 1, 64, "dense", FAR),
    (64, 4, 16, "dense", PI), (64, 4, 24, "rows", FAR), (64, 4, 32, "rows", {}), (64, 12, 16, "dense", FAR),
    (64, 12, 48, "rows", NEAR),
])
def test_many_units_per_share_bf16(D, G, page, layout, geo):
    run(torch.bfloat16, D, G, 8, page, LENS, geo, layout, seed=300 + G, tiles=24 if D == 64 else 32)


@pytest.mark.parametrize("D,G,page,layout,geo", [
    (128, 1, 16, "dense", {}), (128, 2, 24, "dense", PI), (128, 4, 64, "rows", FAR), (128, 8, 16, "dense", NEAR),
    (128, 3, 7, "rows", {}), (64, 1, 64, "dense", FAR), (64, 2, 16, "rows", NEAR), (64, 4, 24, "dense", PI), (64, 7, 16, "dense", {}),
])
def test_many_tiles_per_share_f32(D, G, page, layout, geo):
    run(torch.float32, D, G, 4, page, [40007, 0, 30001, 20000, 9999, 3], geo, layout, seed=320 + G, tiles=16)


@pytest.mark.parametrize("lens", [[40000], [70001, 17], [1, 33333]])
@pytest.mark.parametrize("D,G,page,layout,geo", [
    (128, 4, 64, "dense", {}), (128, 4, 16, "rows", FAR), (128, 12, 128, "dense", PI), (128, 9, 24, "dense", NEAR),
    (128, 16, 16, "rows", {}), (64, 4, 16, "rows", PI), (64, 16, 64, "dense", FAR), (64, 10, 24, "dense", {}),
])
def test_joins_inside_a_block(D, G, page, layout, geo, lens):
    """Few segments cut into many shares: neighbouring shares' partials become one in the block."""
    hk = 8
    w_most, _, gt = shares(torch.bfloat16, D, G, lens, hk)
    blocks = SMS * (2 if D == 64 and gt == 8 else 1)
    units = sum(-(-n // 16) for n in lens) * hk * -(-G // gt)
    assert w_most > 16 * len(lens) * hk * -(-G // gt) and min(w_most, units // 2) > 3 * blocks
    run(torch.bfloat16, D, G, hk, page, lens, geo, layout, seed=340 + G)


@pytest.mark.parametrize("D,G", [(128, 4), (128, 12), (64, 4), (64, 12)])
def test_queries_at_odd_addresses(D, G):
    """A slice that begins on a 2-byte boundary, sequences an odd number of elements apart."""
    hk, lens = 2, [3001, 0, 500]
    g = torch.Generator("cuda").manual_seed(360)
    flat = (torch.randn((3 * (hk * G * D + 3) + 1,), generator=g, device="cuda") * 0.4).bfloat16()
    q = flat[1:].as_strided((3, hk * G, D), (hk * G * D + 3, D, 1), 1)
    assert q.data_ptr() % 4 == 2 and q.stride(0) % 2 == 1
    run(torch.bfloat16, D, G, hk, 16, lens, {}, seed=361, q=q, tiles=0)
    odd = flat[:3 * hk * G * D].reshape(3, hk * G, D)
    wide = torch.zeros((3, hk * G, D + 1), dtype=torch.bfloat16, device="cuda")
    wide[..., :D] = odd
    run(torch.bfloat16, D, G, hk, 16, lens, {}, seed=361, q=wide[..., :D], tiles=0)


@pytest.mark.parametrize("dtype,lens,page,G", [(torch.bfloat16, [50000, 700, 0, 20011], 16, 4), (torch.bfloat16, [9000, 30000], 24, 12),
                                               (torch.float32, [20000, 33, 7001], 16, 4)])
def test_a_sequence_alone_and_beside_others(dtype, lens, page, G):
    """The shares' borders follow the whole batch, so the last bits of a sequence may depend on the
    others; within the tolerances it does not: alone and beside others are both as defined."""
    D, hk = 128, 4
    c = make(lens, hk, D, page, dtype, 370, "dense")
    g = torch.Generator("cuda").manual_seed(371)
    q = (torch.randn((len(lens), hk * G, D), generator=g, device="cuda") * 0.4).to(dtype)
    geo = Geometry(inv_freq(D).cuda())
    cache = paged.PagedCache(c["k"], c["v"], c["table"], c["lens"])
    together = paged.decode(q, cache, geo)
    assert torch.equal(together, paged.decode(q, cache, geo))  # the same batch: the same bits
    for b, n in enumerate(lens):
        alone = paged.decode(q[b:b + 1], cache.with_pages(c["table"][b:b + 1], c["lens"][b:b + 1]), geo)[0]
        if n == 0:
            assert not alone.any() and not together[b].any()
            continue
        want, _, mag, size = definition(q, c, b, geo.inv_freq)
        ds = (3 * 2.0 ** -16 if dtype is torch.bfloat16 else 0.0) + (D + 64) * 2.0 ** -24
        steps = max(2, *(shares(dtype, D, G, x, hk)[1] for x in (lens, [n])))
        depth = (2 if dtype is torch.bfloat16 else 8) * steps + 1776 / 4 + 64
        tol = U[dtype] * want.abs() + (1 + U[dtype]) * (torch.expm1(2 * ds * size) + depth * 2.0 ** -22 + 2.0 ** -16) * mag
        for got in (alone, together[b]):
            assert ((got.double() - want).abs() <= tol).all()
