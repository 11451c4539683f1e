"""float64 restatements of the speculative-step operators (tests only)."""

from __future__ import annotations

import math

import torch


def norm_rope(x, weight, cos_sin, positions, *, eps, interleaved):
    """x [B,T,H,D] -> (rotated rows float64, largest |normalised element| of each row [B,T,H,1])."""
    x = x.double()
    y = x
    if weight is not None:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    out = torch.zeros_like(y)
    r = cos_sin.shape[1]
    for b in range(x.shape[0]):
        for t in range(x.shape[1]):
            pos = int(positions[b, t])
            if not 0 <= pos < cos_sin.shape[0]:
                continue
            out[b, t] = y[b, t]
            c, s = cos_sin[pos, : r // 2].double(), cos_sin[pos, r // 2:].double()
            for i in range(r // 2):
                lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
                out[b, t, :, lo] = y[b, t, :, lo] * c[i] - y[b, t, :, hi] * s[i]
                out[b, t, :, hi] = y[b, t, :, hi] * c[i] + y[b, t, :, lo] * s[i]
    return out, y.abs().amax(-1, keepdim=True)


def write_rows(cache, rows, table, slots, live):
    """Rows [B,T,Hkv,D] into the pages of `cache`, in place."""
    bs = cache.shape[1]
    for b in range(rows.shape[0]):
        for t in range(rows.shape[1]):
            s = int(slots[b, t])
            if not bool(live[b, t]) or not 0 <= s < table.shape[1] * bs:
                continue
            page = int(table[b, s // bs])
            if 0 <= page < cache.shape[0]:
                cache[page, s % bs] = rows[b, t]


def tree_decode(q, k_cache, v_cache, table, lens, mask, drafts, scale=None):
    """-> (out float64, sum p |v| / sum p of each output), both [B,T,Hq,D]."""
    b_, t_, hq, d = q.shape
    hkv = k_cache.shape[2]
    g = hq // hkv
    bs = k_cache.shape[1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(b_):
        n_keys = min(max(int(lens[b]), 0), table.shape[1] * bs)
        n = t_ if drafts is None else min(max(int(drafts[b]), 0), t_)
        if n_keys == 0:
            continue
        pages = table[b, : (n_keys + bs - 1) // bs].long()
        k = k_cache[pages].flatten(0, 1)[:n_keys].double()
        v = v_cache[pages].flatten(0, 1)[:n_keys].double()
        prefix = n_keys - n
        for i in range(n):
            bits = ((1 << (i + 1)) - 1) if mask is None else int(mask[b, i]) & (2**64 - 1)
            seen = [t for t in range(n_keys) if t < prefix or (bits >> (t - prefix)) & 1]
            if not seen:
                continue
            kk, vv = k[seen], v[seen]
            for h in range(hq):
                s = (kk[:, h // g] @ q[b, i, h].double()) * scale
                p = torch.softmax(s, 0)
                out[b, i, h] = p @ vv[:, h // g]
                mag[b, i, h] = p @ vv[:, h // g].abs()
    return out, mag


def compact(cache, table, src, dst):
    bs = cache.shape[1]
    cap = table.shape[1] * bs

    def at(b, pos):
        if not 0 <= pos < cap:
            return None
        page = int(table[b, pos // bs])
        return (page, pos % bs) if 0 <= page < cache.shape[0] else None

    new = cache.clone()
    for b in range(src.shape[0]):
        for i in range(src.shape[1]):
            frm, to = at(b, int(src[b, i])), at(b, int(dst[b]) + i)
            if frm is not None and to is not None:
                new[to] = cache[frm]
    return new


def copy_pages(cache, src, dst):
    new = cache.clone()
    for i, j in zip(src.tolist(), dst.tolist()):
        if 0 <= i < cache.shape[0] and 0 <= j < cache.shape[0]:
            new[j] = cache[i]
    return new


def norm_rope_rows(x, weight, cos_sin, positions, *, eps, interleaved):
    """`norm_rope` for many tokens at once."""
    x = x.double()
    y = x if weight is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    r = cos_sin.shape[1]
    pos = positions.long()
    live = ((pos >= 0) & (pos < cos_sin.shape[0]))[:, :, None, None]
    angles = cos_sin.double()[pos.clamp(0, cos_sin.shape[0] - 1)][:, :, None]
    c, s = angles[..., : r // 2], angles[..., r // 2:]
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    out = y.clone()
    out[..., lo] = y[..., lo] * c - y[..., hi] * s
    out[..., hi] = y[..., hi] * c + y[..., lo] * s
    return torch.where(live, out, torch.zeros_like(out)), y.abs().amax(-1, keepdim=True)


def tree_decode_rows(q, k_cache, v_cache, table, lens, mask, drafts, scale=None):
    """`tree_decode` with all rows of a sequence and kv head at once."""
    b_, t_, hq, d = q.shape
    hkv, bs = k_cache.shape[2], k_cache.shape[1]
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(b_):
        n_keys = min(max(int(lens[b]), 0), table.shape[1] * bs)
        n = t_ if drafts is None else min(max(int(drafts[b]), 0), t_)
        if n_keys == 0 or n == 0:
            continue
        pages = table[b, : (n_keys + bs - 1) // bs].long()
        k = k_cache[pages].flatten(0, 1)[:n_keys].double().transpose(0, 1)      # [hkv, keys, d]
        v = v_cache[pages].flatten(0, 1)[:n_keys].double().transpose(0, 1)
        number = torch.arange(n_keys) - (n_keys - n)                            # of the drafted token
        if mask is None:
            seen = number[None] <= torch.arange(n)[:, None]
        else:
            seen = (number[None] < 0) | ((mask[b, :n, None] >> number.clamp(0, 63)[None]) & 1).bool()
        rows = q[b, :n].double().view(n, hkv, g, d).permute(1, 2, 0, 3)         # [hkv, g, n, d]
        s = torch.einsum("hgnd,hkd->hgnk", rows, k) * scale
        s = s.masked_fill(~seen, -math.inf)
        any_seen = seen.any(1)[:, None]
        p = torch.where(any_seen, torch.softmax(s, -1), torch.zeros_like(s))
        out[b, :n] = torch.einsum("hgnk,hkd->nhgd", p, v).reshape(n, hq, d)
        mag[b, :n] = torch.einsum("hgnk,hkd->nhgd", p, v.abs()).reshape(n, hq, d)
    return out, mag
