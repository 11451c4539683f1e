"""Measured cases of the operators of a speculative decoding step over the paged KV cache.

``qk_norm_rope`` / ``qk_norm_rope_append`` normalise and rotate queries and keys (and write keys
and values into their pages), ``gqa_tree_decode`` attends for a tree of drafted tokens,
``kv_compact`` moves the accepted path together in the cache and ``kv_copy_pages`` copies pages of
sequences that fork.  ``run`` computes an operator in its plain form where ``own`` is false and
calls the library where it is true.
"""

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6
_DEV = "cuda"


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # one new token of each of 64 sequences, on its way into the cache before a decode step
        dict(name="rope_append_b64", op="rope_append", batch=64, tokens=1, q_heads=32, kv_heads=8, head_dim=128,
             rot_dim=128, block_size=16, dtype="bf16", len_lo=1024, len_hi=4096, interleaved=False, ragged=False,
             fused_qkv=True),
        # the drafted tokens of a speculative step, ragged, interleaved pairs, slices of one projection's output
        dict(name="rope_append_tree", op="rope_append", batch=16, tokens=16, q_heads=28, kv_heads=4, head_dim=128,
             rot_dim=128, block_size=16, dtype="fp16", len_lo=256, len_hi=2048, interleaved=True, ragged=True,
             fused_qkv=True),
        # the queries and keys of a dense prefill
        dict(name="rope_prefill", op="rope", batch=4, tokens=4096, q_heads=64, kv_heads=8, head_dim=128, rot_dim=128,
             dtype="bf16", interleaved=False, fused_qkv=False),
        # one short conversation, eight drafted tokens: latency
        dict(name="tree_one_short", op="tree", batch=1, tokens=8, q_heads=32, kv_heads=8, head_dim=128, block_size=16,
             dtype="bf16", len_lo=400, len_hi=400, ragged=False),
        # an ordinary serving batch, eight drafted tokens each
        dict(name="tree_batch", op="tree", batch=64, tokens=8, q_heads=32, kv_heads=8, head_dim=128, block_size=16,
             dtype="bf16", len_lo=1024, len_hi=4096, ragged=False),
        # groups of seven heads, sixteen drafted tokens at most, some sequences with fewer
        dict(name="tree_ragged", op="tree", batch=32, tokens=16, q_heads=28, kv_heads=4, head_dim=128, block_size=16,
             dtype="fp16", len_lo=256, len_hi=2048, ragged=True),
        # long contexts, wide trees: 256 query rows for each key and value head
        dict(name="tree_long", op="tree", batch=4, tokens=32, q_heads=64, kv_heads=8, head_dim=128, block_size=32,
             dtype="bf16", len_lo=32768, len_hi=131072, ragged=False),
        # the 32-bit configuration
        dict(name="tree_fp32", op="tree", batch=4, tokens=4, q_heads=32, kv_heads=8, head_dim=128, block_size=16,
             dtype="fp32", len_lo=64, len_hi=512, ragged=False),
        # the accepted path of a few sequences / of a large batch
        dict(name="compact_b8", op="compact", batch=8, accepted=5, kv_heads=8, head_dim=128, block_size=16,
             dtype="bf16", len_lo=64, len_hi=512),
        dict(name="compact_b256", op="compact", batch=256, accepted=16, kv_heads=8, head_dim=128, block_size=16,
             dtype="bf16", len_lo=64, len_hi=512),
        # a fork's last page for a few sequences / a prompt's pages moved to make room
        dict(name="copy_pages_16", op="copy_pages", pages=16, kv_heads=8, head_dim=128, block_size=16, dtype="bf16"),
        dict(name="copy_pages_4096", op="copy_pages", pages=4096, kv_heads=8, head_dim=128, block_size=16,
             dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope_append", "rope", "tree", "tree", "tree", "compact", "copy_pages"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8])
    head_dim = rng.choice([64, 80, 96, 128, 128, 256])
    block_size = rng.choice([8, 16, 16, 32, 64])
    c = dict(op=op, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype)
    if op in ("rope_append", "rope"):
        rot = rng.choice([head_dim, head_dim, head_dim // 2])
        c.update(batch=_log_int(rng, 1, 64), tokens=_log_int(rng, 1, 64 if op == "rope_append" else 1024),
                 q_heads=kv_heads * group, rot_dim=rot, interleaved=rng.random() < 0.5, fused_qkv=rng.random() < 0.5)
        if op == "rope_append":
            lo = _log_int(rng, 64, 1024)
            c.update(block_size=block_size, len_lo=lo, len_hi=lo + _log_int(rng, 1, 1024), ragged=rng.random() < 0.5)
        return c
    if op == "tree":
        batch = _log_int(rng, 1, 64)
        tokens = _log_int(rng, 1, 8 if dtype == "fp32" else 64)
        # no more tokens than the long listed case, and few 32-bit ones
        most = min(32768, (4096 if dtype == "fp32" else 262144) // batch)
        hi = _log_int(rng, 64, max(65, most))
        lo = max(tokens, _log_int(rng, 1, hi))
        c.update(batch=batch, tokens=tokens, q_heads=kv_heads * group, block_size=block_size, len_lo=lo,
                 len_hi=max(lo, hi), ragged=rng.random() < 0.5)
        return c
    if op == "compact":
        lo = _log_int(rng, 64, 256)
        c.update(batch=_log_int(rng, 1, 256), accepted=_log_int(rng, 1, 33), block_size=block_size, len_lo=lo,
                 len_hi=lo + _log_int(rng, 1, 256))
        return c
    c.update(pages=_log_int(rng, 1, 1024), block_size=block_size)
    return c


# --------------------------------------------------------------------------- the inputs
def _lengths(case, gen):
    """Context lengths spread evenly over the case's range, in an order drawn from the seed."""
    b, lo, hi = case["batch"], case["len_lo"], case["len_hi"]
    lens = lo + ((torch.arange(b, dtype=torch.float64) + 0.5) * ((hi - lo) / b)).to(torch.int64)
    return lens[torch.randperm(b, generator=gen)]


def _table(lens, bs, gen):
    """(int32 page table with -1 in unused places, number of pages): pages in random order, the last one spare."""
    used = (lens + bs - 1) // bs
    need = int(used.sum())
    width = max(1, int(used.max()))
    perm = torch.randperm(need, generator=gen)
    cols = torch.arange(width).expand(len(lens), width)
    live = cols < used[:, None]
    table = torch.full((len(lens), width), -1, dtype=torch.int64)
    table[live] = perm
    return table.to(torch.int32).to(_DEV), need + 1


def _normal(shape, dtype, dgen):
    return torch.empty(shape, dtype=_DT[dtype], device=_DEV).normal_(generator=dgen)


def _draft_lens(case, gen):
    t = case["tokens"]
    if not case["ragged"]:
        return torch.full((case["batch"],), t, dtype=torch.int64)
    return torch.randint(1, t + 1, (case["batch"],), generator=gen)


def _tree(case, gen):
    """Parents of each drafted token (-1: the prefix), and every token's depth."""
    b, t = case["batch"], case["tokens"]
    parent = torch.full((b, t), -1, dtype=torch.int64)
    depth = torch.zeros((b, t), dtype=torch.int64)
    for i in range(1, t):
        parent[:, i] = torch.randint(max(0, i - 6), i, (b,), generator=gen)
        depth[:, i] = depth.gather(1, parent[:, i:i + 1]).squeeze(1) + 1
    return parent, depth


def _mask_bits(parent):
    b, t = parent.shape
    bits = torch.zeros((b, t), dtype=torch.int64)
    for i in range(t):
        up = bits.gather(1, parent[:, i:i + 1].clamp(min=0)).squeeze(1)
        one = 1 << i if i < 63 else -(1 << 63)
        bits[:, i] = torch.where(parent[:, i] >= 0, up, torch.zeros_like(up)) | one
    return bits


def _rope_table(n, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], dim=1).to(torch.float32).to(_DEV)


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dgen = torch.Generator(device=_DEV).manual_seed(seed)
    op, dt, hkv, d = case["op"], case["dtype"], case["kv_heads"], case["head_dim"]
    s = dict(op=op)
    if op in ("rope", "rope_append"):
        b, t, hq = case["batch"], case["tokens"], case["q_heads"]
        nv = hkv if op == "rope_append" else 0
        if case["fused_qkv"]:
            qkv = _normal((b, t, hq + hkv + nv, d), dt, dgen)
            s.update(q=qkv[:, :, :hq], k=qkv[:, :, hq:hq + hkv], v=qkv[:, :, hq + hkv:])
        else:
            s.update(q=_normal((b, t, hq, d), dt, dgen), k=_normal((b, t, hkv, d), dt, dgen),
                     v=_normal((b, t, nv, d), dt, dgen))
        s["qw"] = (1 + 0.1 * torch.randn(d, generator=dgen, device=_DEV)).to(_DT[dt])
        s["kw"] = (1 + 0.1 * torch.randn(d, generator=dgen, device=_DEV)).to(_DT[dt])
        s["interleaved"] = case["interleaved"]
        if op == "rope":
            s["cos_sin"] = _rope_table(t, case["rot_dim"])
            s["positions"] = torch.arange(t, dtype=torch.int32, device=_DEV).expand(b, t).contiguous()
            return s
        lens = _lengths(case, gen)                       # tokens already in the cache
        n = _draft_lens(case, gen)
        _, depth = _tree(case, gen)
        live = torch.arange(t)[None] < n[:, None]
        slots = lens[:, None] + torch.arange(t)[None]
        pos = lens[:, None] + depth
        table, pages = _table(lens + t, case["block_size"], gen)
        s.update(table=table, k_cache=_normal((pages, case["block_size"], hkv, d), dt, dgen),
                 v_cache=_normal((pages, case["block_size"], hkv, d), dt, dgen),
                 slots=torch.where(live, slots, -1).to(torch.int32).to(_DEV),
                 positions=torch.where(live, pos, -1).to(torch.int32).to(_DEV),
                 cos_sin=_rope_table(case["len_hi"] + t, case["rot_dim"]))
        return s
    if op == "tree":
        b, t, hq = case["batch"], case["tokens"], case["q_heads"]
        lens = _lengths(case, gen).clamp(min=t)          # the drafted tokens are in the cache already
        table, pages = _table(lens, case["block_size"], gen)
        parent, _ = _tree(case, gen)
        s.update(q=_normal((b, t, hq, d), dt, dgen), k_cache=_normal((pages, case["block_size"], hkv, d), dt, dgen),
                 v_cache=_normal((pages, case["block_size"], hkv, d), dt, dgen), table=table,
                 lens=lens.to(torch.int32).to(_DEV), mask=_mask_bits(parent).to(_DEV),
                 drafts=_draft_lens(case, gen).to(torch.int32).to(_DEV))
        return s
    if op == "compact":
        lens = _lengths(case, gen)
        a = case["accepted"]
        table, pages = _table(lens, case["block_size"], gen)
        span = min(64, int(lens.min()))                  # the drafted tokens are the last `span`
        take = min(a, span)
        src = torch.full((case["batch"], a), -1, dtype=torch.int64)
        pick = torch.rand((case["batch"], span), generator=gen).argsort(1)[:, :take].sort(1).values
        count = torch.randint(1, take + 1, (case["batch"],), generator=gen)
        src[:, :take] = torch.where(torch.arange(take)[None] < count[:, None], (lens - span)[:, None] + pick, -1)
        s.update(table=table, k_cache=_normal((pages, case["block_size"], hkv, d), dt, dgen),
                 v_cache=_normal((pages, case["block_size"], hkv, d), dt, dgen), src=src.to(torch.int32).to(_DEV),
                 dst=(lens - span).to(torch.int32).to(_DEV))
        return s
    n = case["pages"]
    perm = torch.randperm(2 * n + 3, generator=gen).to(torch.int32).to(_DEV)
    shape = (2 * n + 3, case["block_size"], hkv, d)
    s.update(k_cache=_normal(shape, dt, dgen), v_cache=_normal(shape, dt, dgen), src=perm[:n].contiguous(),
             dst=perm[n:2 * n].contiguous())
    return s


# --------------------------------------------------------------------------- the plain forms
def _norm_rotate(x, w, cos, sin, live, interleaved):
    """x [B,T,H,D] in 32 bits, normalised for each head and rotated by the angles of its token."""
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
    r = 2 * cos.shape[-1]
    if interleaved:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    y = torch.cat([turned, y[..., r:]], dim=-1)
    return torch.where(live, y, torch.zeros_like(y))


def _plain_rope(s):
    pos = s["positions"].long()
    live = (pos >= 0)[..., None, None]
    cs = s["cos_sin"][pos.clamp(min=0)][:, :, None, :]
    half = cs.shape[-1] // 2
    args = (cs[..., :half], cs[..., half:], live, s["interleaved"])
    q = _norm_rotate(s["q"], s["qw"], *args).to(s["q"].dtype)
    k = _norm_rotate(s["k"], s["kw"], *args).to(s["k"].dtype)
    if s["op"] == "rope":
        return q, k
    bs = s["k_cache"].shape[1]
    slots = s["slots"].long()
    page = s["table"].long().gather(1, (slots.clamp(min=0) // bs))
    spare = s["k_cache"].shape[0] * bs - 1
    row = torch.where(slots >= 0, page * bs + slots.clamp(min=0) % bs, spare).flatten()
    keep = (slots >= 0).flatten()[:, None, None]
    for cache, new in ((s["k_cache"], k), (s["v_cache"], s["v"])):
        flat = cache.flatten(0, 1)
        flat[row] = torch.where(keep, new.flatten(0, 1), flat[spare])
    return q, s["k_cache"], s["v_cache"]


def _plain_tree(s):
    q, table, lens = s["q"], s["table"], s["lens"].long()
    b, t, hq, d = q.shape
    hkv = s["k_cache"].shape[2]
    at = table.long().clamp(min=0)
    k = s["k_cache"][at].flatten(1, 2).float()           # [B, L, Hkv, D]
    v = s["v_cache"][at].flatten(1, 2).float()
    keys = torch.arange(k.shape[1], device=q.device)
    n = s["drafts"].long()[:, None, None]
    prefix = lens[:, None, None] - n
    off = keys[None, None] - prefix                      # number of the drafted token, negative in the prefix
    bit = (s["mask"][:, :, None] >> off.clamp(0, 63)) & 1
    seen = (off < 0) | ((off < n) & (bit == 1))
    seen = seen & (torch.arange(t, device=q.device)[None, :, None] < n)
    seen = seen[:, None, :, None, :].expand(b, 1, t, hq // hkv, -1).flatten(2, 3)
    rows = q.float().view(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    score = rows @ k.permute(0, 2, 3, 1) * (1.0 / math.sqrt(d))
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p @ v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
    return out.view(b, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(q.dtype)


def _plain_compact(s):
    bs = s["k_cache"].shape[1]
    src, table = s["src"].long(), s["table"].long()
    keep = src >= 0
    frm = src.clamp(min=0)
    to = (s["dst"].long()[:, None] + torch.arange(src.shape[1], device=src.device)).clamp(max=table.shape[1] * bs - 1)
    spare = s["k_cache"].shape[0] * bs - 1
    frm = torch.where(keep, table.gather(1, frm // bs) * bs + frm % bs, spare).flatten()
    to = torch.where(keep, table.gather(1, to // bs) * bs + to % bs, spare).flatten()
    for cache in (s["k_cache"], s["v_cache"]):
        flat = cache.flatten(0, 1)
        flat[to] = flat[frm]
    return s["k_cache"], s["v_cache"]


def _plain_copy(s):
    for cache in (s["k_cache"], s["v_cache"]):
        cache[s["dst"].long()] = cache[s["src"].long()]
    return s["k_cache"], s["v_cache"]


def run(s):
    if own:
        import attention_b200 as attn
        if s["op"] == "rope":
            return attn.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos_sin"], s["positions"], eps=_EPS,
                                     interleaved=s["interleaved"])
        if s["op"] == "rope_append":
            q = attn.qk_norm_rope_append(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos_sin"], s["positions"],
                                         s["k_cache"], s["v_cache"], s["table"], slots=s["slots"], eps=_EPS,
                                         interleaved=s["interleaved"])
            return q, s["k_cache"], s["v_cache"]
        if s["op"] == "tree":
            return attn.gqa_tree_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["mask"],
                                        draft_lens=s["drafts"])
        if s["op"] == "compact":
            attn.kv_compact(s["k_cache"], s["v_cache"], s["table"], s["src"], s["dst"])
        else:
            attn.kv_copy_pages(s["k_cache"], s["v_cache"], s["src"], s["dst"])
        return s["k_cache"], s["v_cache"]
    return {"rope": _plain_rope, "rope_append": _plain_rope, "tree": _plain_tree, "compact": _plain_compact,
            "copy_pages": _plain_copy}[s["op"]](s)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size, hkv, d, op = _SIZE[case["dtype"]], case["kv_heads"], case["head_dim"], case["op"]
    if op in ("rope", "rope_append"):
        tokens = case["batch"] * case["tokens"]
        heads = case["q_heads"] + hkv * (2 if op == "rope_append" else 1)
        return {"bytes": tokens * (2 * heads * d * size + 4 * case["rot_dim"] + 8),
                "flops": tokens * (case["q_heads"] + hkv) * (4 * d + 3 * case["rot_dim"])}
    if op == "tree":
        b, t, hq = case["batch"], case["tokens"], case["q_heads"]
        lo, hi = case["len_lo"], case["len_hi"]
        total = sum(max(t, lo + int((i + 0.5) * ((hi - lo) / b))) for i in range(b))
        return {"bytes": 2 * total * hkv * d * size + 2 * b * t * hq * d * size, "flops": 4 * t * hq * d * total}
    row = hkv * d * size
    if op == "compact":
        # on average half of the places hold an accepted token
        rows = case["batch"] * (case["accepted"] + 1) / 2
        return {"bytes": 4 * rows * row, "flops": 0}
    return {"bytes": 4 * case["pages"] * case["block_size"] * row, "flops": 0}


# --------------------------------------------------------------------------- 64 bits
def _exact_rows(x, w, angles_cos, angles_sin, interleaved):
    """Rows of one token [H, D] as complex pairs turned by the token's angles."""
    x = x.double()
    y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS) * w.double()
    r = 2 * angles_cos.shape[-1]
    turn = torch.complex(angles_cos.double(), angles_sin.double()).unsqueeze(-2)
    if interleaved:
        z = torch.view_as_complex(y[..., :r].unflatten(-1, (r // 2, 2)).contiguous()) * turn
        y[..., :r] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * turn
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("rope", "rope_append"):
        pos = s["positions"].cpu().numpy()
        half = case["rot_dim"] // 2
        q = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
        k = torch.zeros(s["k"].shape, dtype=torch.float64, device=_DEV)
        for b in range(case["batch"]):
            rows = torch.from_numpy(np.flatnonzero(pos[b] >= 0)).to(_DEV)
            cs = s["cos_sin"].index_select(0, s["positions"][b].index_select(0, rows).long())
            for out, x, w in ((q, s["q"], s["qw"]), (k, s["k"], s["kw"])):
                out[b, rows] = _exact_rows(x[b].index_select(0, rows), w, cs[:, :half], cs[:, half:],
                                           case["interleaved"])
        if op == "rope":
            return q, k
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        slots, table = s["slots"].cpu().numpy(), s["table"].cpu().numpy()
        bs = case["block_size"]
        for b in range(case["batch"]):
            for i in np.flatnonzero(slots[b] >= 0):
                page, line = int(table[b, slots[b, i] // bs]), int(slots[b, i] % bs)
                kc[page, line] = k[b, i]
                vc[page, line] = s["v"][b, i].double()
        return q, kc, vc
    if op == "tree":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
        lens, drafts = s["lens"].tolist(), s["drafts"].tolist()
        masks = s["mask"].tolist()
        bs, d = case["block_size"], case["head_dim"]
        group = case["q_heads"] // case["kv_heads"]
        for b, (n_keys, n) in enumerate(zip(lens, drafts)):
            pages = s["table"][b, :(n_keys + bs - 1) // bs].long()
            hide = np.zeros((n, n_keys), dtype=bool)
            for i in range(n):
                for j in range(n):
                    hide[i, n_keys - n + j] = not (masks[b][i] >> j) & 1
            hide = torch.from_numpy(hide).to(_DEV)
            for h in range(case["kv_heads"]):
                k = s["k_cache"][pages, :, h].reshape(-1, d)[:n_keys].double()
                v = s["v_cache"][pages, :, h].reshape(-1, d)[:n_keys].double()
                q = s["q"][b, :n, h * group:(h + 1) * group].double()
                score = torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(d)
                score.masked_fill_(hide[:, None, :], -math.inf)
                weight = torch.softmax(score, dim=-1)
                out[b, :n, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", weight, v)
        return out
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    if op == "compact":
        src, dst, table = s["src"].cpu().numpy(), s["dst"].cpu().numpy(), s["table"].cpu().numpy()
        bs = case["block_size"]
        where = [(int(table[b, src[b, i] // bs]), int(src[b, i] % bs), int(table[b, (dst[b] + i) // bs]),
                  int((dst[b] + i) % bs)) for b, i in zip(*np.nonzero(src >= 0))]
        fp, fl, tp, tl = (torch.tensor(x, device=_DEV) for x in zip(*where))
        for cache in (kc, vc):
            moved = cache[fp, fl].clone()
            cache[tp, tl] = moved
        return kc, vc
    for i, j in zip(s["src"].tolist(), s["dst"].tolist()):
        kc[j], vc[j] = kc[i], vc[i]
    return kc, vc
