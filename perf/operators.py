"""Cases for the operators of the paged key-value cache (``sta.paged``).

    append   raw key / value rows of new tokens written into the pages of their sequences
    decode   attention of one new token per sequence over its pages, keys rotated where they are
             read (plain, position-interpolated, YaRN or Dual Chunk Attention geometry), on
             request with the attention weight of every key added to the cache's weights
    evict    the keys with the largest accumulated weight (and always the first ``sinks`` and the
             last ``recent`` ones) copied into fresh pages, in order: a key's slot is its new position

``run`` computes a case in elementary torch operations, or, where ``own`` is true, through the
framework.  A cache is (pages, kv heads, page size, head dim); a sequence's slot j lies in page
``table[b, j // page size]``.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
#: bytes of keys and values that the largest case holds in reach of one call
_MOST = 1 * 8 * 131072 * 128 * 2 * 2


def _case(op, **kw):
    d = dict(op=op, dtype="bf16", batch=1, heads=32, kv_heads=8, dim=128, page=64, length=1024,
             ragged=False)
    if op == "decode":
        d.update(theta=5e5, pos_scale=1.0, rope_scale=1.0, chunk=0, window=0, weights=False)
    elif op == "append":
        d.update(rows=1)
    else:
        d.update(budget=512, sinks=32, recent=32)
    d.update(kw)
    return d


def listed():
    return [
        # a chat's next token early in its context, nothing else on the GPU: latency
        _case("decode", name="decode_short", length=1000, page=16),
        # one sequence at the 32k context of a grouped-query layer with YaRN (factor 4)
        _case("decode", name="decode_yarn_32k", length=32768, rope_scale=1.1386294361119891),
        # a serving batch of conversations of every age, with the weights that eviction needs
        _case("decode", name="decode_batch_weights", batch=32, length=8192, page=16, ragged=True,
              weights=True),
        # the longest context, one sequence: the whole card on eight kv heads
        _case("decode", name="decode_128k", length=131072, page=128),
        # two long sequences in Dual Chunk Attention positions (chunk 6144, local window 1024)
        _case("decode", name="decode_dca_64k", batch=2, length=65536, chunk=6144, window=1024),
        # every q head with a kv head of its own, positions interpolated by 1/2, odd page size
        _case("decode", name="decode_mha_pi", batch=2, heads=32, kv_heads=32, length=8191, page=24,
              theta=1e4, pos_scale=0.5, weights=True),
        # single precision, head dim 64, a small ragged batch
        _case("decode", name="decode_f32", batch=8, dtype="f32", heads=4, kv_heads=4, dim=64, length=4096, page=16,
              ragged=True, theta=1e4),
        # the step of a serving batch: one token of each of 64 sequences
        _case("append", name="append_step", batch=64, length=8192, page=16, ragged=True),
        # prompts of two sequences stored after their prefill
        _case("append", name="append_prompts", batch=2, length=16, rows=32768, ragged=True),
        # one sequence over its budget: latency
        _case("evict", name="evict_one", length=1536, page=16, budget=1024),
        # a batch of sequences cut back to the selection cap of 2048 keys, single precision
        _case("evict", name="evict_batch_f32", batch=16, dtype="f32", length=8192, page=16, ragged=True, budget=2048),
        # long prompts reduced to their 8192 heaviest keys
        _case("evict", name="evict_long", batch=4, length=65536, budget=8192),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("decode", "decode", "append", "evict"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    dim = rng.choice((64, 128))
    group = rng.choice((1, 2, 3, 4, 6, 8, 16))
    kv = rng.choice((1, 2, 4, 8)) if group > 1 else rng.choice((2, 4, 8, 32))
    batch = _log(rng, 1, 64)
    room = _MOST // (kv * dim * (4 if dtype == "f32" else 2) * 2 * batch)
    base = dict(dtype=dtype, dim=dim, kv_heads=kv, heads=kv * group, batch=batch,
                page=rng.choice((1, 8, 16, 16, 24, 32, 64, 128, 256)), ragged=batch > 1 and rng.random() < 0.8)
    base["page"] = max(base["page"], 8 if room > 4096 else 1)
    if op == "decode":
        c = _case(op, **base, length=_log(rng, 1, min(131072, room)), weights=rng.random() < 0.4,
                  theta=rng.choice((1e4, 5e5)), pos_scale=rng.choice((1.0, 1.0, 0.5, 0.125)),
                  rope_scale=rng.choice((1.0, 1.1386294361119891)))
        if rng.random() < 0.25:
            c.update(chunk=rng.choice((320, 1280, 6144)), window=64, pos_scale=1.0)
            c["window"] = 1024 if c["chunk"] == 6144 else 64
        return c
    if op == "append":
        return _case(op, **base, length=_log(rng, 1, min(16384, max(1, room // 2))),
                     rows=1 if rng.random() < 0.5 else _log(rng, 2, min(32768, max(2, room // 2))))
    length = _log(rng, 64, min(65536, max(64, room // 2)))
    return _case(op, **base, length=length, budget=rng.randint(8, length), sinks=rng.choice((0, 4)), recent=rng.choice((0, 1, 4)))


def _lengths(case, top, zero):
    """The sequences' lengths: `top` all, or spread from short to `top` (a batch slot without a sequence has none)."""
    b = case["batch"]
    if not case["ragged"] or b == 1:
        return [top] * b
    r = random.Random(1009 * b + top)
    n = [max(1, int(top * r.random() ** 1.5)) for _ in range(b)]
    n[r.randrange(b)] = top
    if zero and b >= 4:
        n[n.index(min(n))] = 0
    return n


def _plan(case):
    """Lengths now, rows to append, and the slots that each sequence's pages have to hold."""
    if case["op"] == "append":
        lens = _lengths(case, case["length"], True)
        rows = [1] * case["batch"] if case["rows"] == 1 else _lengths(case, case["rows"], False)
        return lens, rows, [a + b for a, b in zip(lens, rows)]
    lens = _lengths(case, case["length"], case["op"] == "decode")
    return lens, [0] * case["batch"], lens


def _pages(n, page):
    return (n + page - 1) // page


def prepare(case, seed):
    dev, g = "cuda", torch.Generator("cuda").manual_seed(seed)
    dt, D, P, B, hk, H = _TYPES[case["dtype"]], case["dim"], case["page"], case["batch"], case["kv_heads"], case["heads"]
    lens, rows, slots = _plan(case)
    used = [_pages(n, P) for n in slots]
    fresh = [_pages(min(n, case["budget"]), P) for n in lens] if case["op"] == "evict" else []
    pages = sum(used) + sum(fresh) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32).cpu()

    def table(counts, at):
        t = torch.full((B, max(1, max(counts))), -1, dtype=torch.int32)  # -1: no page
        for b, n in enumerate(counts):
            t[b, :n] = order[at:at + n]
            at += n
        return t.to(dev)

    # noise plus a common low-rank part, as the framework's synthetic inputs have: some keys stand out
    mix = torch.randn((16, D), generator=g, device=dev) * 0.5

    def filled(shape, common):
        x = torch.empty(shape + (D,), dtype=dt, device=dev)
        for part in x.split(max(1, (1 << 26) // max(1, x[0].numel()))):
            y = torch.randn(part.shape, generator=g, device=dev)
            if common:
                y += torch.randn(part.shape[:-1] + (16,), generator=g, device=dev) @ mix
            part.copy_(y)
        return x

    s = {"case": case, "k": filled((pages, hk, P), True), "v": filled((pages, hk, P), False),
         "table": table(used, 0), "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    if case["op"] == "decode":
        s["q"] = filled((B, H), True)
        inv = 1.0 / (case["theta"] ** (torch.arange(0, D, 2, dtype=torch.float32) / D))
        s["inv_freq"] = inv.to(dev)
        if case["weights"]:  # what a few dozen earlier steps left
            s["weights"] = 4 * torch.rand((pages, hk, P), generator=g, device=dev) ** 4
            s["weights_out"] = torch.zeros_like(s["weights"])
    elif case["op"] == "append":
        n = max(rows)
        s["k_new"] = filled((B, n, hk), True).transpose(1, 2)  # as a projection leaves them
        s["v_new"] = filled((B, n, hk), False).transpose(1, 2)
        s["counts"] = None if n == 1 else torch.tensor(rows, dtype=torch.int32, device=dev)
        s["weights"] = torch.rand((pages, hk, P), generator=g, device=dev)
        s["lens_out"] = torch.zeros_like(s["lens"])
    else:
        w = torch.exp(2 * torch.randn((pages, hk, P), generator=g, device=dev) - 4)
        # keys that no query has looked at yet tie at zero, and quantised ones tie elsewhere
        u = torch.rand((pages, hk, P), generator=g, device=dev)
        w = torch.where(u < 0.1, torch.zeros_like(w), torch.where(u < 0.3, (w * 64).round() / 64, w))
        s["weights"] = w
        s["table_out"] = table(fresh, sum(used))
    if own:
        _calls(s)
    return s


def _calls(s):
    """The handles that a program keeps: the caches over the tensors, and the geometry."""
    c = s["case"]
    paged, core = _framework()
    w = s.get("weights")
    s["cache"] = paged.PagedCache(s["k"], s["v"], s["table"], s["lens"], weights=w)
    if c["op"] == "decode":
        dca = (c["chunk"], c["window"]) if c["chunk"] else None
        s["geometry"] = core.Geometry(s["inv_freq"], c["pos_scale"], c["rope_scale"], dca)


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-thresholded-attention_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from sta import core, paged
    return paged, core


def run(s):
    c = s["case"]
    if c["op"] == "append":
        if own:
            _framework_append(s)
        else:
            _append(s)
        return {"k": s["k"], "v": s["v"], "weights": s["weights"], "lens": s["lens_out"]}
    if c["op"] == "decode":
        out = _framework_decode(s) if own else _decode(s)
        return {"out": out, "weights": s["weights_out"]} if c["weights"] else {"out": out}
    lens, kept = _framework_evict(s) if own else _evict(s)
    return {"k": s["k"], "v": s["v"], "weights": s["weights"], "lens": lens, "kept": kept}


def _framework_append(s):
    paged = sys.modules["sta.paged"]
    paged.append(s["cache"], s["k_new"], s["v_new"], counts=s["counts"], lens_out=s["lens_out"])


def _framework_decode(s):
    paged = sys.modules["sta.paged"]
    return paged.decode(s["q"], s["cache"], s["geometry"], weights_out=s.get("weights_out"))


def _framework_evict(s):
    paged, c = sys.modules["sta.paged"], s["case"]
    after, kept = paged.evict(s["cache"], c["budget"], s["table_out"], n_global=c["sinks"], n_local=c["recent"])
    return after.lens, kept


# ---- plain forms ------------------------------------------------------------------------------
def _append(s):
    lens, n, P = s["lens"].long(), s["k_new"].shape[2], s["k"].shape[2]
    i = torch.arange(n, device=lens.device)
    counts = torch.full_like(lens, n) if s["counts"] is None else s["counts"].long()
    b, r = (i[None, :] < counts[:, None]).nonzero(as_tuple=True)
    j = lens[b] + r
    page, slot = s["table"][b, j // P].long(), j % P
    s["k"][page, :, slot] = s["k_new"][b, :, r]
    s["v"][page, :, slot] = s["v_new"][b, :, r]
    s["weights"][page, :, slot] = 0.0
    s["lens_out"].copy_(lens + counts)


def _dense(pool, table):
    """(pages, heads, page size, ...) -> (batch, heads, slots, ...) in 32 bits; a missing page reads page 0."""
    x = pool[table.clamp(min=0).long()].transpose(1, 2)
    return x.reshape(x.shape[:2] + (-1,) + x.shape[4:]).float()


def _rotated(x, pos, inv_freq, scale):
    """Rows x (..., n, D) at positions pos (..., n): angles in 64 bits, products in 32."""
    a = pos[..., None] * inv_freq.double()
    c, s = (a.cos() * scale).float(), (a.sin() * scale).float()
    x1, x2 = x.chunk(2, dim=-1)
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)


def _decode(s):
    c = s["case"]
    B, hk, D, P = c["batch"], c["kv_heads"], c["dim"], c["page"]
    inv, scale, L = s["inv_freq"], c["rope_scale"], c["chunk"] - c["window"]
    k, v = _dense(s["k"], s["table"]), _dense(s["v"], s["table"])
    lens = s["lens"].long()
    j = torch.arange(k.shape[2], device=k.device)
    last = (lens - 1).clamp(min=0)
    q = s["q"].float().reshape(B, hk, -1, D)

    def scores(query_pos, keys):
        at = query_pos.double()[:, None, None].expand(q.shape[:3])
        return _rotated(q, at, inv, scale) @ keys.transpose(-1, -2)

    if c["chunk"]:
        keys = _rotated(k, (j % L).double(), inv, scale)
        away = (last // L)[:, None, None, None] - j // L
        same = scores(last % L, keys)
        before = scores((L + last % L).clamp(max=c["chunk"]), keys)
        older = scores(torch.full_like(last, min(2 * L - 1, c["chunk"])), keys)
        x = torch.where(away == 0, same, torch.where(away == 1, before, older))
    else:
        keys = _rotated(k, j.double() * c["pos_scale"], inv, scale)
        x = scores(last * c["pos_scale"], keys)
    seen = (j < lens[:, None])[:, None, None, :]
    x = (x * (1.0 / math.sqrt(D))).masked_fill(~seen, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)  # a sequence of length 0 gives zeros
    out = (p @ v).reshape(B, -1, D).to(s["q"].dtype)
    if c["weights"]:
        w = p.sum(dim=2).reshape(B, hk, -1, P).transpose(1, 2)  # (batch, table width, heads, page size)
        b, t = (torch.arange(w.shape[1], device=w.device) * P < lens[:, None]).nonzero(as_tuple=True)
        page = s["table"][b, t].long()
        mine = seen.reshape(B, -1, 1, P)[b, t]
        s["weights_out"][page] = torch.where(mine, s["weights"][page] + w[b, t], s["weights_out"][page])
    return out


def _evict(s):
    c = s["case"]
    P, budget, hk = c["page"], c["budget"], c["kv_heads"]
    lens = s["lens"].long()
    w = _dense(s["weights"], s["table"])
    j = torch.arange(w.shape[2], device=w.device)
    at = lens[:, None, None]
    w = torch.where((j < c["sinks"]) | (j >= at - c["recent"]), torch.full_like(w, math.inf), w)
    w = torch.where(j < at, w, torch.full_like(w, -math.inf))
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]
    new = lens.clamp(max=budget)
    r = torch.arange(order.shape[-1], device=w.device)
    kept = torch.where(r < new[:, None, None], order, torch.full_like(order, w.shape[2])).sort(dim=-1).values
    b, h, r = (r < new[:, None, None]).expand(kept.shape).nonzero(as_tuple=True)
    src = kept[b, h, r]
    page, slot = s["table"][b, src // P].long(), src % P
    to, to_slot = s["table_out"][b, r // P].long(), r % P
    for x in (s["k"], s["v"], s["weights"]):
        x[to, h, to_slot] = x[page, h, slot]
    out = torch.full((c["batch"], hk, budget), -1, dtype=torch.int32, device=w.device)
    out[b, h, r] = src.to(torch.int32)
    return new.to(torch.int32), out


# ---- the definition in 64 bits -------------------------------------------------------------------
def _slots(table_row, n, page):
    """Page and offset of a sequence's slots 0 .. n-1."""
    j = torch.arange(n, device=table_row.device)
    return table_row.long().repeat_interleave(page)[:n], j.remainder(page)


def exact(case, seed):
    s = prepare(case, seed)
    lens, rows, _ = _plan(case)
    P, B, hk, D = case["page"], case["batch"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        k, v, w = s["k"].double(), s["v"].double(), s["weights"].double()
        for b in range(B):
            page, off = (x[lens[b]:] for x in _slots(s["table"][b], lens[b] + rows[b], P))
            k[page, :, off] = s["k_new"][b].double().transpose(0, 1)[:rows[b]]
            v[page, :, off] = s["v_new"][b].double().transpose(0, 1)[:rows[b]]
            w[page, :, off] = 0
        return {"k": k, "v": v, "weights": w, "lens": torch.tensor([a + b for a, b in zip(lens, rows)], dtype=torch.int32)}
    if case["op"] == "evict":
        k, v, w = s["k"].double(), s["v"].double(), s["weights"].double()
        kept = torch.full((B, hk, case["budget"]), -1, dtype=torch.int32)
        for b in range(B):
            page, off = _slots(s["table"][b], lens[b], P)
            n = min(lens[b], case["budget"])
            to, to_off = _slots(s["table_out"][b], n, P)
            here = s["weights"][page, :, off].t().double()  # (heads, keys)
            here[:, :case["sinks"]] = 1e300
            here[:, max(0, lens[b] - case["recent"]):] = 1e300
            keep = torch.argsort(-here, dim=-1, stable=True)[:, :n].sort(dim=-1).values
            for h in range(hk):
                for new, old in ((k, s["k"]), (v, s["v"]), (w, s["weights"])):
                    new[to, h, to_off] = old[page[keep[h]], h, off[keep[h]]].double()
            kept[b, :, :n] = keep.cpu().int()
        return {"k": k, "v": v, "weights": w, "lens": torch.tensor([min(n, case["budget"]) for n in lens], dtype=torch.int32), "kept": kept}
    inv = s["inv_freq"].double()
    out = torch.zeros((B, case["heads"], D), dtype=torch.float64, device="cuda")
    w = s["weights_out"].double() if case["weights"] else None
    L, half, group = case["chunk"] - case["window"], D // 2, case["heads"] // hk

    def turn(x, pos):  # complex rotation: (x1 + i x2) e^(i pos f)
        z = torch.complex(x[..., :half], x[..., half:])
        return z * torch.polar(torch.full_like(pos[:, None] * inv, case["rope_scale"]), pos[:, None] * inv)

    for b in range(B):
        n = lens[b]
        if n == 0:
            continue
        page, off = _slots(s["table"][b], n, P)
        j = torch.arange(n, device="cuda")
        i = n - 1
        if case["chunk"]:
            key_pos = j.remainder(L)
            away = i // L - torch.div(j, L, rounding_mode="floor")
            far = [i % L, min(L + i % L, case["chunk"]), min(2 * L - 1, case["chunk"])]
            query_pos = torch.tensor(far, device="cuda")[away.clamp(max=2)]
        else:
            key_pos, query_pos = j * case["pos_scale"], torch.full((n,), i * case["pos_scale"], device="cuda", dtype=torch.float64)
        places, which = query_pos.double().unique(return_inverse=True)  # the query's positions, three at most
        for h in range(hk):
            z = turn(s["k"][page, h, off].double(), key_pos.double())
            for m in range(h * group, (h + 1) * group):
                turned = turn(s["q"][b, m].double()[None], places)
                x = (z @ turned.conj().t()).real.gather(1, which[:, None])[:, 0]
                p = torch.softmax(x / math.sqrt(D), dim=0)
                out[b, m] = p @ s["v"][page, h, off].double()
                if w is not None:
                    first = m == h * group
                    w[page, h, off] = p + (s["weights"][page, h, off].double() if first else w[page, h, off])
    return {"out": out, "weights": w} if case["weights"] else {"out": out}


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    row = case["kv_heads"] * case["dim"] * es * 2  # key and value of one token
    lens, rows, slots = _plan(case)
    B = case["batch"]
    small = 4 * (sum(_pages(n, case["page"]) for n in slots) + B)
    if case["op"] == "append":
        n = sum(rows)
        return {"bytes": n * (2 * row + 4 * case["kv_heads"]) + small + 4 * B, "flops": 0}
    n = sum(lens)
    if case["op"] == "decode":
        bytes_ = n * row + 2 * B * case["heads"] * case["dim"] * es + small
        if case["weights"]:
            bytes_ += 8 * n * case["kv_heads"]
        return {"bytes": bytes_, "flops": 4 * n * case["heads"] * case["dim"]}
    m = sum(min(x, case["budget"]) for x in lens)
    over = sum(x for x in lens if x > case["budget"])
    return {"bytes": m * (2 * row + 8 * case["kv_heads"]) + 4 * over * case["kv_heads"]
            + 4 * B * case["kv_heads"] * case["budget"] + small, "flops": 0}
