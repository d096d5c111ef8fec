"""The paged cache's operators from their definitions, in 64 bits on the CPU (for the tests)."""
import math

import torch


def make(batch_lens, *, hk, D, page, dtype, seed, spare=3, width=0, scale=1.0, garbage=None):
    """A pool with a random page order, tables and lengths; slots past a length hold `garbage`."""
    g = torch.Generator().manual_seed(seed)
    used = [max(0, -(-n // page)) for n in batch_lens]
    n_pages = sum(used) + spare
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(batch_lens), max([1, width] + used)), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    k = (torch.randn((n_pages, hk, page, D), generator=g) * scale).to(dtype)
    v = torch.randn((n_pages, hk, page, D), generator=g).to(dtype)
    w = torch.rand((n_pages, hk, page), generator=g)
    if garbage is not None:
        live = torch.zeros((n_pages, page), dtype=torch.bool)
        for b, n in enumerate(batch_lens):
            for j in range(n):
                live[table[b, j // page], j % page] = True
        for x in (k, v):
            x.transpose(1, 2)[~live] = garbage
    lens = torch.tensor(batch_lens, dtype=torch.int32)
    return dict(k=k, v=v, table=table, lens=lens, weights=w, free=order[at:])


def rows(pool, table_row, n, page):
    """Slots 0 .. n-1 of one sequence: (heads, n, ...)."""
    j = torch.arange(n)
    return pool[table_row.long()[j // page], :, j % page].transpose(0, 1)


def rotate(x, pos, inv_freq, rope_scale):
    a = pos.double()[:, None] * inv_freq.double()
    c, s = a.cos() * rope_scale, a.sin() * rope_scale
    x1, x2 = x.double().chunk(2, -1)
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), -1)


def decode(q, c, inv_freq, pos_scale=1.0, rope_scale=1.0, dca=None, sm_scale=None):
    """(out, per sequence attention weights (H, n), bound): float64.  `bound` (B, H, D) is the sum
    of p |v| and `size` (B, H) the largest sum of |q_i k_i| * scale, for the tolerances."""
    B, H, D = q.shape
    page, hk = c["k"].shape[2], c["k"].shape[1]
    G = H // hk
    sm = 1.0 / math.sqrt(D) if sm_scale is None else sm_scale
    out = torch.zeros((B, H, D), dtype=torch.float64)
    mag = torch.zeros((B, H, D), dtype=torch.float64)
    size = torch.zeros((B, H), dtype=torch.float64)
    probs = []
    for b in range(B):
        n = int(c["lens"][b])
        p_b = torch.zeros((H, n), dtype=torch.float64)
        if n:
            k, v = rows(c["k"], c["table"][b], n, page), rows(c["v"], c["table"][b], n, page).double()
            j, i = torch.arange(n), n - 1
            if dca is None:
                kp, qp = j * pos_scale, torch.full((n,), i * pos_scale, dtype=torch.float64)
            else:
                s, w = dca
                Lc = s - w
                kp, away = j % Lc, i // Lc - j // Lc
                qp = torch.where(away == 0, i % Lc, torch.where(away == 1, min(Lc + i % Lc, s), min(2 * Lc - 1, s))).double()
            for h in range(H):
                kr = rotate(k[h // G], kp, inv_freq, rope_scale)
                qr = rotate(q[b, h].expand(n, D), qp, inv_freq, rope_scale)
                x = (kr * qr).sum(-1) * sm
                size[b, h] = (kr.norm(dim=-1) * qr.norm(dim=-1)).max() * sm
                p_b[h] = torch.softmax(x, 0)
                out[b, h] = p_b[h] @ v[h // G]
                mag[b, h] = p_b[h] @ v[h // G].abs()
        probs.append(p_b)
    return out, probs, mag, size


def added_weights(c, probs, base):
    """weights_out after one decode: base plus each key's attention weight."""
    out = base.double().clone()
    page, hk = c["k"].shape[2], c["k"].shape[1]
    for b, p in enumerate(probs):
        n = p.shape[1]
        j = torch.arange(n)
        got = p.reshape(hk, p.shape[0] // hk, n).sum(1)
        out[c["table"][b].long()[j // page], :, j % page] += got.t()
    return out


def evict(c, budget, n_global, n_local):
    """Kept slots (B, hk, budget) int32, -1 beyond, by sorting (weight descending, slot ascending)."""
    B, hk, page = c["table"].shape[0], c["k"].shape[1], c["k"].shape[2]
    kept = torch.full((B, hk, budget), -1, dtype=torch.int32)
    for b in range(B):
        n = int(c["lens"][b])
        w = rows(c["weights"][..., None], c["table"][b], n, page)[..., 0] if n else torch.zeros((hk, 0))
        for h in range(hk):
            forced = [j for j in range(n) if j < n_global or j >= n - n_local]
            val = [-math.inf if math.isnan(x) else float(x) for x in w[h]]
            nan = [math.isnan(x) for x in w[h]]
            rest = sorted((j for j in range(n) if not (j < n_global or j >= n - n_local)),
                          key=lambda j: (nan[j], -val[j], j))
            keep = sorted(range(n) if n <= budget else forced + rest[:budget - len(forced)])
            kept[b, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
    return kept
