"""The operators around a tree of drafted tokens: norm + rotation (+ append), tree attention,
compaction, page copies; each against float64, then a whole step.

Tolerances.  h(t) is half a step of a type relative to the value: finfo(t).eps / 2.
* norm + rotation: one rounding, h |y|, after an fp32 chain.  Its longest path is a sum of at most
  256 squares (8 in a lane, 5 shuffles: 13 roundings), a division, a reciprocal square root (2 steps
  each), two products and a fused rotation: below 24 roundings of 2^-24, relative to the pair, whose
  size is at most sqrt(2) times the row's largest element m: 24 * 1.42 * 2^-24 < 2.1e-6 m.
* tree attention: out = sum p v / sum p with A = sum p |v| / sum p.  A score is an fp32 sum of D
  products, off by at most D 2^-23 |q| |k| scale; p is off by that (twice: its sum too), the exp by
  2^-21 and, in the 16-bit kernels, by a rounding h(t) of p; sums over L keys by L 2^-23 of A; then
  one rounding of the result.
  For random values with zero mean the errors are independent and so is their size: a rounding has
  an rms of h / sqrt(3) of its value, and sum(p dv)^2 relates to sum (p v)^2 as p's error to p, so
  the relative error of a whole sequence (2-norm) stays under h(t) (two roundings: sqrt(2/3) h) plus
  the fp32 terms.  A forgotten or wrongly seen key among L changes it by about 1/sqrt(L).
"""

import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import attention_b200 as attn
from attention_b200 import _cabi, synth
from oracle import speculative_oracle as ref

gpu = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_wait_ran_out(request):
    """After every GPU test: no bounded wait of the tensor-core kernel gave up."""
    yield
    if "gpu" in request.keywords and torch.cuda.is_available():
        assert attn.speculative.tree_tc_status() == 0


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half of the smallest step near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rope_table(n, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def check_rope(got, x, w, cs, pos, eps, interleaved):
    want, m = ref.norm_rope(x, w, cs, pos, eps=eps, interleaved=interleaved)
    tol = half_step(x.dtype) * want.abs() + 2.1e-6 * m + smallest(x.dtype)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.double() - want).abs() <= tol).all()


# --------------------------------------------------------------------------- norm and rotation
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (256, 256), (128, 64), (128, 24), (80, 80), (96, 48), (5, 2),
                                   (1, 0), (200, 200), (256, 0), (8, 8)])
def test_norm_rope_against_float64(dtype, interleaved, d, rot):
    gen = torch.Generator().manual_seed(d * 7 + rot)
    b, t, hq, hkv = 2, 5, 6, 3
    q = torch.randn(b, t, hq, d, generator=gen).to(dtype)
    k = (3 * torch.randn(b, t, hkv, d, generator=gen)).to(dtype)
    qw, kw = (1 + 0.2 * torch.randn(2, d, generator=gen)).to(dtype)
    cs = rope_table(40, rot)
    pos = torch.randint(0, 40, (b, t), generator=gen, dtype=torch.int32)
    pos[1, 2], pos[0, 4] = -1, 40                       # padding on either side of the table
    dq, dk = q.to(DEV), k.to(DEV)
    args = (qw.to(DEV), kw.to(DEV), cs.to(DEV), pos.to(DEV))
    qo, ko = attn.qk_norm_rope(dq, dk, *args, eps=1e-5, interleaved=interleaved)
    check_rope(qo.cpu(), q, qw, cs, pos, 1e-5, interleaved)
    check_rope(ko.cpu(), k, kw, cs, pos, 1e-5, interleaved)
    assert torch.count_nonzero(qo[1, 2]) == 0 and torch.count_nonzero(ko[0, 4]) == 0
    assert torch.equal(dq.cpu(), q) and torch.equal(dk.cpu(), k)
    # in place
    a, c = attn.qk_norm_rope(dq, dk, *args, eps=1e-5, interleaved=interleaved, q_out=dq, k_out=dk)
    assert a is dq and c is dk and torch.equal(dq, qo) and torch.equal(dk, ko)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ["fused", "offset", "head_strided", "no_weight", "fp32_weight", "three_dims", "expanded"])
def test_norm_rope_layouts_and_weights(dtype, case):
    gen = torch.Generator().manual_seed(3)
    b, t, hq, hkv, d = 3, 4, 5, 2, 128
    qkv = torch.randn(b, t, hq + 2 * hkv, d, generator=gen).to(dtype).to(DEV)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hkv]
    w = (1 + 0.2 * torch.randn(2, d, generator=gen)).to(dtype)
    cs = rope_table(64, d)
    pos = torch.randint(0, 64, (b, t), generator=gen, dtype=torch.int32)
    if case == "offset":                                # not 16-byte aligned
        flat = torch.empty(q.numel() + 1, dtype=dtype, device=DEV)
        qo = flat[1:].view(q.shape)
        qo.copy_(q)
        q = qo
    if case == "head_strided":                          # [B, H, T, D] in memory
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
    if case == "expanded":                              # one row for every head
        k = k[:, :, :1].expand(b, t, hkv, d)
    if case == "fp32_weight":
        w = w.float() + 1e-4
    qw, kw = (None, None) if case == "no_weight" else (w[0].to(DEV), w[1].to(DEV))
    if case == "three_dims":
        a, c = attn.qk_norm_rope(q[:, 1], k[:, 1], qw, kw, cs.to(DEV), pos[:, 1].contiguous().to(DEV))
        a, c, q, k, pos = a[:, None], c[:, None], q[:, 1:2], k[:, 1:2], pos[:, 1:2]
    else:
        a, c = attn.qk_norm_rope(q, k, qw, kw, cs.to(DEV), pos.to(DEV))
    assert a.is_contiguous() and c.is_contiguous()
    check_rope(a.cpu(), q.cpu(), None if qw is None else w[0], cs, pos, 1e-6, False)
    check_rope(c.cpu(), k.cpu(), None if qw is None else w[1], cs, pos, 1e-6, False)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,bs,hq,hkv,t", [(128, 16, 8, 2, 1), (128, 5, 28, 4, 7), (64, 1, 3, 3, 16), (80, 8, 10, 5, 3),
                                           (37, 6, 2, 1, 4), (256, 32, 16, 8, 9)])
def test_append_writes_pages_and_nothing_else(dtype, d, bs, hq, hkv, t):
    gen = torch.Generator().manual_seed(d + bs)
    b, pages = 4, 3
    pool = b * pages + 2
    q = torch.randn(b, t, hq, d, generator=gen).to(dtype)
    k, v = torch.randn(2, b, t, hkv, d, generator=gen).to(dtype)
    kc, vc = torch.randn(2, pool, bs, hkv, d, generator=gen).to(dtype)
    qw, kw = (1 + 0.2 * torch.randn(2, d, generator=gen)).to(dtype)
    rot = d // 2 * 2
    cs = rope_table(100, rot)
    table = torch.randperm(pool, generator=gen)[: b * pages].view(b, pages).to(torch.int32)
    table[1, 1], table[2, 0] = -1, pool                 # pages outside the pool
    cap = pages * bs
    slots = torch.stack([torch.randperm(max(cap, t), generator=gen)[:t] for _ in range(b)]).to(torch.int32)
    slots[0, 0] = -3
    slots[3, t - 1] = cap
    pos = torch.randint(0, 100, (b, t), generator=gen, dtype=torch.int32)
    pos[3, 0] = -1                                      # padding: no write either
    dk, dv = kc.to(DEV), vc.to(DEV)
    out = attn.qk_norm_rope_append(q.to(DEV), k.to(DEV), v.to(DEV), qw.to(DEV), kw.to(DEV), cs.to(DEV), pos.to(DEV), dk,
                                   dv, table.to(DEV), slots=slots.to(DEV))
    check_rope(out.cpu(), q, qw, cs, pos, 1e-6, False)
    dense = attn.qk_norm_rope(q.to(DEV), k.to(DEV), qw.to(DEV), kw.to(DEV), cs.to(DEV), pos.to(DEV))
    assert torch.equal(out, dense[0])
    live = (pos >= 0) & (pos < 100)
    ref.write_rows(kc, dense[1].cpu(), table, slots, live)      # (the keys themselves: tested above)
    ref.write_rows(vc, v, table, slots, live)
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)


@gpu
def test_append_defaults_its_slots_to_the_positions_and_takes_one_token():
    gen = torch.Generator().manual_seed(1)
    b, hq, hkv, d, bs = 3, 8, 2, 128, 16
    q = torch.randn(b, hq, d, generator=gen).half().to(DEV)
    k, v = torch.randn(2, b, hkv, d, generator=gen).half().to(DEV)
    kc = torch.zeros(6, bs, hkv, d, dtype=torch.float16, device=DEV)
    vc = torch.zeros_like(kc)
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([3, 16, 31], dtype=torch.int32, device=DEV)
    cs = rope_table(32, d).to(DEV)
    out = attn.qk_norm_rope_append(q, k, v, None, None, cs, pos, kc, vc, table, out=q)
    assert out is q
    for i, (page, line) in enumerate([(0, 3), (3, 0), (5, 15)]):
        assert torch.equal(vc[page, line], v[i])
    assert int(torch.count_nonzero(vc.abs().sum((2, 3)))) == 3


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot,offset", [(128, 128, 0), (128, 64, 1), (5, 4, 0), (96, 12, 0)])
def test_empty_angle_table_makes_every_token_padding(dtype, interleaved, d, rot, offset):
    """No position lies inside a table of no rows: zeros come back, nothing is read from it and nothing written.
    (`offset` 1, and sizes that are no multiples of 8, take the kernel for rows of any alignment.)"""
    gen = torch.Generator().manual_seed(d)
    b, t, hq, hkv = 2, 3, 4, 2
    flat = torch.randn(b * t * hq * d + offset, generator=gen).to(dtype).to(DEV)
    q = flat[offset:].view(b, t, hq, d)
    k, v = torch.randn(2, b, t, hkv, d, generator=gen).to(dtype).to(DEV)
    w = torch.ones(d, dtype=dtype, device=DEV)
    cs = torch.empty(0, rot, device=DEV)
    pos = torch.tensor([[0, -1, 5], [2**31 - 1, -2**31, 1]], dtype=torch.int32, device=DEV)
    a, c = attn.qk_norm_rope(q, k, w, w, cs, pos, interleaved=interleaved)
    assert torch.count_nonzero(a) == 0 and torch.count_nonzero(c) == 0
    kc, vc = torch.randn(2, 4, 8, hkv, d, generator=gen).to(dtype).to(DEV)
    keep = kc.clone(), vc.clone()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    slots = torch.arange(t, dtype=torch.int32, device=DEV).repeat(b, 1)
    a = attn.qk_norm_rope_append(q, k, v, w, w, cs, pos, kc, vc, table, slots=slots, interleaved=interleaved)
    assert torch.count_nonzero(a) == 0
    assert torch.equal(kc, keep[0]) and torch.equal(vc, keep[1])


# --------------------------------------------------------------------------- tree attention
def tree_case(lengths, t, hq, hkv, d, bs, dtype, seed=0, drafts=None, masks="tree"):
    gen = torch.Generator().manual_seed(seed)
    lens = torch.tensor(lengths, dtype=torch.int32)
    b = len(lengths)
    pool = max(1, sum((n + bs - 1) // bs for n in lengths)) + 2
    q = torch.randn(b, t, hq, d, generator=gen).to(dtype)
    k, v = torch.randn(2, pool, bs, hkv, d, generator=gen).to(dtype)
    table = synth.build_block_table(lens, bs, pool, gen)
    mask = None
    if masks == "tree":
        rows = []
        for _ in range(b):
            bits = []
            for i in range(t):
                par = int(torch.randint(-1, i, (1,), generator=gen)) if i else -1
                x = (bits[par] if par >= 0 else 0) | (1 << i)
                bits.append(x)
            rows.append([x - (1 << 64) if x >= 1 << 63 else x for x in bits])
        mask = torch.tensor(rows, dtype=torch.int64)
    elif masks == "random":
        mask = torch.randint(-(2**63), 2**63 - 1, (b, t), generator=gen)
    dl = None if drafts is None else torch.tensor(drafts, dtype=torch.int32)
    return q, k, v, table, lens, mask, dl


def on_gpu(*ts):
    return tuple(None if x is None else x.to(DEV) for x in ts)


def check_tree(got, case, scale=None):
    q, k, v, table, lens, mask, dl = case
    want, mag = ref.tree_decode(q, k, v, table, lens, mask, dl, scale)
    d, dtype = q.shape[-1], q.dtype
    h = half_step(dtype)
    sc = 1 / math.sqrt(d) if scale is None else scale
    size = sc * float(q.double().norm(dim=-1).max()) * float(k.double().norm(dim=-1).max())
    fp32 = 2 * d * 2.0**-23 * size + 2.0**-20 + int(lens.max()) * 2.0**-23
    p_round = 0.0 if dtype == torch.float32 else h
    got = got.cpu().double()
    tol = h * want.abs() + (p_round + fp32) * mag + smallest(dtype)
    assert ((got - want).abs() <= tol).all()
    for b in range(q.shape[0]):
        norm = float(want[b].norm())
        assert float((got[b] - want[b]).norm()) <= (h + fp32) * norm


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,hq,hkv", [(1, 8, 8), (1, 8, 2), (3, 5, 5), (8, 8, 2), (16, 14, 2), (33, 8, 1), (64, 4, 2),
                                      (9, 64, 4), (3, 130, 1), (2, 128, 1), (20, 15, 1), (43, 6, 2)])
def test_tree_heads_and_tokens(dtype, t, hq, hkv, kernel):
    case = tree_case([t, 70 + t, 300, 129], t, hq, hkv, 128, 16, dtype, seed=t)
    dc = on_gpu(*case)
    check_tree(attn.gqa_tree_decode(*dc[:6], draft_lens=dc[6], kernel=kernel), case)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,bs", [(128, 1), (64, 5), (96, 24), (80, 16), (40, 16), (8, 8), (256, 32), (200, 64), (37, 7),
                                  (1, 16), (128, 8), (64, 128), (128, 256), (256, 8), (72, 16), (136, 384), (24, 32)])
def test_tree_head_dims_and_pages(dtype, d, bs):
    case = tree_case([5, 64, 257], 5, 6, 2, d, bs, dtype, seed=d)
    dc = on_gpu(*case)
    for kernel in ("auto", "simt"):
        check_tree(attn.gqa_tree_decode(*dc[:6], kernel=kernel), case)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,hq", [(2, 4), (5, 4), (9, 6)])
@pytest.mark.parametrize("d", [2, 50, 66, 100, 130, 202, 255])
def test_tree_rows_that_are_not_whole_16_byte_pieces(dtype, t, hq, d):
    case = tree_case([t + 1, 150, 64, 97], t, hq, 2, d, 16, dtype, seed=d)
    check_tree(attn.gqa_tree_decode(*on_gpu(*case[:6])), case)


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_lengths_and_draft_counts(dtype, kernel):
    """Empty sequences, one key, fewer keys than drafted tokens, no drafted token, tile and page edges."""
    lengths = [0, 1, 3, 16, 127, 128, 129, 255, 256, 257, 40, 50]
    drafts = [6, 6, 6, 0, 1, 6, 6, 2, 6, 5, -4, 99]
    for masks in ("tree", "random", None):
        case = tree_case(lengths, 6, 8, 2, 128, 16, dtype, seed=5, drafts=drafts, masks=masks)
        dc = on_gpu(*case)
        got = attn.gqa_tree_decode(*dc[:6], draft_lens=dc[6], kernel=kernel)
        check_tree(got, case)
        assert torch.count_nonzero(got[0]) == 0 and torch.count_nonzero(got[3]) == 0
        assert torch.count_nonzero(got[4, 1:]) == 0 and torch.count_nonzero(got[10]) == 0


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_rows_that_see_nothing_and_hidden_infinities(dtype, kernel):
    """A mask of zero with no prefix is an empty row; what is hidden may be infinite or NaN."""
    t, d, bs = 8, 128, 16
    lengths = [t, t + 20, 140, 300]
    case = tree_case(lengths, t, 8, 2, d, bs, dtype, seed=6)
    q, k, v, table, lens, _, _ = case
    mask = torch.full((4, t), 0b1010, dtype=torch.int64)        # tokens 1 and 3 only
    mask[0, 2] = 0                                              # nothing: no prefix either
    mask[1, 2] = 0                                              # the prefix alone
    clean = (q, k.clone(), v.clone(), table, lens, mask, None)
    bad = [float("nan"), float("inf"), float("-inf")]
    k, v = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        for j in (0, 2, 4, 5, 6, 7):                            # hidden from every row
            pos = n - t + j
            page, line = int(table[b, pos // bs]), pos % bs
            k[page, line], v[page, line] = bad[j % 3], bad[(j + b) % 3]
        for pos in range(n, (n + bs - 1) // bs * bs):           # behind the end
            page = int(table[b, pos // bs])
            k[page, pos % bs], v[page, pos % bs] = bad[pos % 3], bad[(pos + 1) % 3]
    dq, dk, dv, dt, dl, dm, _ = on_gpu(q, k, v, table, lens, mask, None)
    got = attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm, kernel=kernel)
    check_tree(got, clean)
    assert torch.count_nonzero(got[0, 2]) == 0
    assert torch.equal(got, attn.gqa_tree_decode(dq, *on_gpu(clean[1], clean[2]), dt, dl, dm, kernel=kernel))


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_infinite_value_reaches_exactly_the_rows_that_see_it(dtype, kernel):
    t, hq, hkv, d, bs = 6, 4, 2, 64, 16
    case = tree_case([200, 40], t, hq, hkv, d, bs, dtype, seed=7)
    q, k, v, table, lens, mask, _ = case
    seen = (mask >> 2) & 1                                      # who sees drafted token 2
    v = v.clone()
    for b, n in enumerate([200, 40]):
        pos = n - t + 2
        v[int(table[b, pos // bs]), pos % bs, 1, 5] = float("inf")
    got = attn.gqa_tree_decode(*on_gpu(q, k, v, table, lens, mask), kernel=kernel).cpu()
    hit = torch.isinf(got) & (got > 0)
    want = torch.zeros_like(hit)
    want[:, :, hq // 2:, 5] = (seen == 1)[:, :, None]
    assert torch.equal(hit, want)
    assert torch.isfinite(got[~want]).all()


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [17.5, 20.0])
@pytest.mark.parametrize("t,hq,d,bs", [(4, 4, 128, 16), (5, 20, 64, 16), (40, 8, 128, 16), (4, 4, 256, 16), (4, 4, 128, 24)])
def test_tree_probabilities_far_below_a_dominating_key(dtype, kernel, nats, t, hq, d, bs):
    """One key far above the others whose value is zero: the result is what the others weigh, e^-nats each.
    In bf16 a rounded probability is off by h(t) of itself down to 2^-126.  In fp16 it is so down to the
    smallest normal number, and below that off by at most half a step of 2^-24; the tensor-core kernel keeps
    the row's largest at 2^11 or more, so relative to the largest that is 2^-25 / 2^11 = 2^-36 for a key, |v| 2^-36
    in the result."""
    lengths = [2500, 300, 1000]
    q, k, v, table, lens, mask, _ = tree_case(lengths, t, hq, 2, d, bs, dtype, seed=t)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    v = 256 * v.abs()
    for b in range(len(lengths)):
        page, line = int(table[b, 77 // bs]), 77 % bs
        k[page, line] = 0.0
        k[page, line, :, 0] = nats * math.sqrt(d) / 8.0
        v[page, line] = 0.0
    got = attn.gqa_tree_decode(*on_gpu(q, k, v, table, lens, mask), kernel=kernel).cpu().double()
    want, mag = ref.tree_decode(q, k, v, table, lens, mask, None)
    h = half_step(dtype)
    size = float(q.double().norm(dim=-1).max()) * float(k.double().norm(dim=-1).max()) / math.sqrt(d)
    fp32 = 2 * d * 2.0**-23 * size + 2.0**-20 + max(lengths) * 2.0**-23
    p_round = 0.0 if dtype == torch.float32 else h
    lowest = 2.0**-36 * max(lengths) * float(v.double().max()) if dtype == torch.float16 else 0.0
    assert ((got - want).abs() <= h * want.abs() + (p_round + fp32) * mag + lowest + smallest(dtype)).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [0.0, 10.0, 1500.0, 3000.0, 6000.0])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("t,hq,d,bs", [(4, 4, 64, 16), (40, 8, 64, 16), (16, 8, 128, 16), (4, 4, 256, 16), (4, 4, 64, 24)])
def test_tree_probabilities_stay_in_range_whatever_the_scores(dtype, size, sign, t, hq, d, bs):
    """Scores of up to 2^26 that differ by a few units (a step of fp32 is 4 there), and a value that is the same for
    every key: the weighted mean is that value.  What the weights are does not matter, but a probability
    must not overflow its type.  Their rounding is off by h(t), below fp16's normal numbers by 2^-25 where the largest
    is 4 at least (the reference may be off by a step): 2^-27 a key."""
    lengths = [600, 77, 300]
    gen = torch.Generator().manual_seed(7)
    q, k, v, table, lens, mask, _ = tree_case(lengths, t, hq, 2, d, bs, dtype, seed=t)
    q, k = 0 * q, 0 * k
    q[..., 0], k[..., 0] = 60000.0, sign * size * math.sqrt(d) / 8.0
    q[..., 1] = 8.0
    k[..., 1] = (torch.rand(k.shape[:-1], generator=gen) * 20).to(dtype)
    v = v[:1, :1].expand(v.shape).contiguous()
    got = attn.gqa_tree_decode(*on_gpu(q, k, v, table, lens, mask)).cpu().double()
    want = v[0, 0].double().repeat_interleave(hq // 2, 0).expand(got.shape)
    p_round = 0.0 if dtype == torch.float32 else half_step(dtype)
    rel = half_step(dtype) + p_round + max(lengths) * 2.0**-23 + 2.0**-20 + max(lengths) * 2.0**-27
    assert ((got - want).abs() <= rel * want.abs() + smallest(dtype)).all()


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(300, 3, 4, 2), (2, 7, 64, 64), (1, 64, 16, 2), (5, 20, 40, 8), (1, 1, 1, 1)])
def test_tree_work_split_over_runs(dtype, kernel, shape):
    """Sequences cut over several runs, many sequences per run, more kv heads than a round holds."""
    b, t, hq, hkv = shape
    gen = torch.Generator().manual_seed(b)
    top = 200 if b > 5 else 900
    lengths = [int(x) for x in torch.randint(0, top, (b,), generator=gen)]
    lengths[0] = 1500 if b < 300 else 700
    case = tree_case(lengths, t, hq, hkv, 64, 16, dtype, seed=b)
    if b == 300:                                                # (the float64 loop over 300 x 3 x 4 rows is slow)
        keep = [0, 1, 2, 127, 128, 129, 255, 256, 257, 298, 299]
    else:
        keep = list(range(b))
    dc = on_gpu(*case)
    got = attn.gqa_tree_decode(*dc[:6], kernel=kernel).cpu()
    q, k, v, table, lens, mask, _ = case
    rows = torch.tensor(keep)
    if t * hq > 400:                                            # compare a few heads
        group = hq // hkv
        heads = [0, hkv - 1]
        cols = torch.tensor([h * group + g for h in heads for g in range(group)])
        k, v = k[:, :, heads].contiguous(), v[:, :, heads].contiguous()
        q, got = q[:, :, cols], got[:, :, cols]
    check_tree(got[rows], (q[rows], k, v, table[rows], lens[rows], mask[rows], None))
    again = attn.gqa_tree_decode(*dc[:6], kernel=kernel).cpu()
    assert torch.equal(again if t * hq <= 400 else again[:, :, cols], got)


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [5, 128, 256, 257, 600, 768, 769, 1030])
def test_tree_of_one_short_sequence(dtype, n, d):
    """One run without a merge up to six tiles, a run a tile behind; infinite drafted values in both."""
    t = 5
    q, k, v, table, lens, mask, _ = case = tree_case([n], t, 6, 2, d, 16, dtype, seed=n)
    check_tree(attn.gqa_tree_decode(*on_gpu(*case[:6])), case)
    v = v.clone()
    pos = n - t + 2
    v[int(table[0, pos // 16]), pos % 16, 1, d - 1] = float("inf")
    got = attn.gqa_tree_decode(*on_gpu(q, k, v, table, lens, mask)).cpu()
    seen = ((mask[0] >> 2) & 1) == 1
    want = torch.zeros(got.shape, dtype=torch.bool)
    want[0, :, 3:, d - 1] = seen[:, None]
    assert torch.equal(torch.isinf(got), want) and torch.isfinite(got[~want]).all()


@gpu
def test_tree_of_one_token_is_the_ordinary_decode_and_a_chain_needs_no_mask():
    case = tree_case([90, 400, 33], 1, 8, 2, 128, 16, torch.bfloat16, seed=2, masks=None)
    dq, dk, dv, dt, dl, _, _ = on_gpu(*case)
    one = attn.gqa_decode(dq[:, 0].contiguous(), dk, dv, dt, dl)
    got = attn.gqa_tree_decode(dq, dk, dv, dt, dl)[:, 0]
    # both within two roundings of the same value; A is at most max |v|
    assert (one.float() - got.float()).abs().max() <= 4 * half_step(torch.bfloat16) * float(dv.float().abs().max())
    case = tree_case([90, 400, 33], 5, 8, 2, 128, 16, torch.bfloat16, seed=2, masks=None)
    dq, dk, dv, dt, dl, _, _ = on_gpu(*case)
    chain = torch.tensor([[(2 << i) - 1 for i in range(5)]] * 3, device=DEV)
    assert torch.equal(attn.gqa_tree_decode(dq, dk, dv, dt, dl), attn.gqa_tree_decode(dq, dk, dv, dt, dl, chain))


@gpu
@pytest.mark.parametrize("scale", [0.03, 1.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_scale_unaligned_rows_out_and_workspace(dtype, scale):
    case = tree_case([100, 17, 260], 4, 8, 2, 64, 16, dtype, seed=9)
    dq, dk, dv, dt, dl, dm, _ = on_gpu(*case)
    flat = torch.empty(dq.numel() + 1, dtype=dtype, device=DEV)
    q_off = flat[1:].view(dq.shape)
    q_off.copy_(dq)
    out = torch.full_like(dq, float("nan"))
    need = attn.tree_workspace_bytes(3, 4, 8, 2, 64, 16, dt.shape[1])
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    assert attn.gqa_tree_decode(q_off, dk, dv, dt, dl, dm, scale=scale, out=out, workspace=ws) is out
    check_tree(out, case, scale)
    check_tree(attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm, scale=scale), case, scale)
    with pytest.raises(RuntimeError, match="workspace"):
        attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm, workspace=ws[256:])
    with pytest.raises(RuntimeError, match="overlap"):
        attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm, out=dq)


@gpu
def test_tree_bad_page_ids_read_some_valid_page():
    case = tree_case([100, 60], 4, 8, 2, 64, 16, torch.float16, seed=9)
    dq, dk, dv, dt, dl, dm, _ = on_gpu(*case)
    dt[0, 1], dt[0, 3], dt[1, 0] = -7, 2**31 - 1, dk.shape[0]
    for kernel in ("auto", "simt"):
        assert torch.isfinite(attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm, kernel=kernel)).all()


@gpu
def test_tree_two_graphs_and_two_streams_share_nothing():
    """Two captured calls and an eager one, replayed at once on streams of their own."""
    cases = [tree_case([1500 + 64 * i, 900], 8, 32, 8, 128, 16, torch.bfloat16, seed=i) for i in range(3)]
    dcs = [on_gpu(*c) for c in cases]
    want = [attn.gqa_tree_decode(*dc[:6]) for dc in dcs]
    graphs, outs = [], []
    for dc in dcs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attn.gqa_tree_decode(*dc[:6]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = attn.gqa_tree_decode(*dcs[2][:6])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])
    # the lengths are read when the graph runs
    dcs[0][4].copy_(torch.tensor([700, 0], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], attn.gqa_tree_decode(*dcs[0][:6]))


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
def test_tree_many_short_and_few_long_pieces_again_and_again(kernel):
    """Chains of a CTA drift apart over many short sequences; the same bits every time."""
    gen = torch.Generator().manual_seed(4)
    for t, hq, hkv, d in [(2, 8, 4, 128), (7, 8, 4, 128), (20, 8, 2, 64), (40, 8, 2, 128)]:
        lengths = [int(x) for x in torch.randint(t, 700, (90,), generator=gen)]
        dq, dk, dv, dt, dl, dm, _ = on_gpu(*tree_case(lengths, t, hq, hkv, d, 16, torch.bfloat16, seed=t))
        want = attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm, kernel=kernel)
        simt = attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm, kernel="simt")
        # both kernels within their roundings of the same value (P and the result; A <= max |v|)
        assert (want.float() - simt.float()).abs().max() <= 3 * half_step(torch.bfloat16) * float(dv.float().abs().max())
        for _ in range(60):
            assert torch.equal(attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm, kernel=kernel), want)


@gpu
def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes per cache and 2^31 elements, pages at its end."""
    bs, hkv, d, t = 16, 8, 256, 4
    pool = 2**31 // (bs * hkv * d) + 40
    gen = torch.Generator().manual_seed(0)
    kc = torch.empty(pool, bs, hkv, d, dtype=torch.bfloat16, device=DEV)
    vc = torch.empty_like(kc)
    lengths = [75, 40]
    lens = torch.tensor(lengths, dtype=torch.int32)
    used = 8
    table = (pool - 1 - torch.arange(2 * used).view(2, used) * 2).to(torch.int32)
    rows = torch.randn(2, 2 * used, bs, hkv, d, generator=gen).bfloat16()
    at = table.flatten().long().to(DEV)
    kc[at], vc[at] = rows[0].to(DEV), rows[1].to(DEV)
    small = torch.arange(2 * used, dtype=torch.int32).view(2, used)
    q = torch.randn(2, t, 16, d, generator=gen).bfloat16()
    for kernel in ("auto", "simt"):
        got = attn.gqa_tree_decode(*on_gpu(q), kc, vc, *on_gpu(table, lens), kernel=kernel)
        check_tree(got, (q, rows[0], rows[1], small, lens, None, None))
    key, val = torch.randn(2, 2, t, hkv, d, generator=gen).bfloat16()
    slots = torch.tensor([[75, 76, 100, 127], [40, 41, 42, 43]], dtype=torch.int32)
    cs = rope_table(200, d)
    dkey = key.to(DEV)
    attn.qk_norm_rope_append(q.to(DEV), dkey, val.to(DEV), None, None, cs.to(DEV), slots.to(DEV), kc, vc, table.to(DEV))
    keys = attn.qk_norm_rope(q.to(DEV), dkey, None, None, cs.to(DEV), slots.to(DEV))[1].cpu()
    live = torch.ones(2, t, dtype=torch.bool)
    ref.write_rows(rows[0], keys, small, slots, live)
    ref.write_rows(rows[1], val, small, slots, live)
    src = torch.tensor([[100, 127, 3], [43, 40, -1]], dtype=torch.int32)
    dst = torch.tensor([75, 40], dtype=torch.int32)
    attn.kv_compact(kc, vc, *on_gpu(table, src, dst))
    want = [ref.compact(r, small, src, dst) for r in rows]
    assert torch.equal(kc[at].cpu(), want[0]) and torch.equal(vc[at].cpu(), want[1])
    frm, to = table[0, :3].to(DEV), (table[0, :3] - 1).to(DEV)
    attn.kv_copy_pages(kc, vc, frm, to)
    assert torch.equal(kc[to.long()], kc[frm.long()]) and torch.equal(vc[to.long()], vc[frm.long()])


@gpu
def test_first_call_of_a_process_may_be_captured():
    """Nothing is looked up or set up in a way that a stream capture forbids."""
    code = """
import sys
sys.path.insert(0, {root!r})
import torch
import attention_b200 as attn
q = torch.randn(2, 4, 8, 128, device="cuda").bfloat16()
kc = torch.randn(9, 16, 2, 128, device="cuda").bfloat16()
vc = torch.randn_like(kc)
table = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
lens = torch.tensor([60, 33], device="cuda", dtype=torch.int32)
cs = torch.randn(64, 128, device="cuda")
pos = torch.tensor([[3, 4, 5, 6], [7, 8, 9, 10]], device="cuda", dtype=torch.int32)
pages = torch.tensor([[0], [8]], device="cuda", dtype=torch.int32)
def step():
    r = attn.qk_norm_rope_append(q, q[:, :, :2], q[:, :, 2:4], None, None, cs, pos, kc, vc, table)
    out = attn.gqa_tree_decode(r, kc, vc, table, lens)
    slow = attn.gqa_tree_decode(r, kc, vc, table, lens, kernel="simt")
    attn.kv_compact(kc, vc, table, pos, lens - 4)
    attn.kv_copy_pages(kc, vc, pages[0], pages[1])
    return r, out, slow
torch.cuda.synchronize()
keep = kc.clone(), vc.clone()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
got = [x.clone() for x in (*got, kc, vc)]
kc.copy_(keep[0]); vc.copy_(keep[1])
want = [*step(), kc, vc]
assert all(torch.equal(a, b) for a, b in zip(got, want))
assert attn.speculative.tree_tc_status() == 0
del g
print("captured")
"""
    root = str(Path(__file__).resolve().parents[1])
    run = subprocess.run([sys.executable, "-c", code.format(root=root)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


# --------------------------------------------------------------------------- moves in the cache
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 16), (1, 5, 3), (3, 37, 1), (2, 64, 7)])
def test_compact_against_reference(dtype, hkv, d, bs):
    gen = torch.Generator().manual_seed(d)
    b, pages, n = 5, 12, 9
    kc, vc = torch.randn(2, b * pages + 1, bs, hkv, d, generator=gen).to(dtype)
    table = torch.randperm(b * pages, generator=gen).view(b, pages).to(torch.int32)
    table[4, 2], table[4, 5] = -1, 10**6
    cap = pages * bs
    src = torch.randint(-1, cap + 2, (b, n), generator=gen, dtype=torch.int32)
    src[0] = torch.arange(n) + 1                        # a shift by one: each source is a destination
    src[1] = torch.arange(n - 1, -1, -1)                # reversed in place
    src[2, 3:6] = 2                                     # the same row often
    dst = torch.tensor([0, 0, 1, cap - 4, 0], dtype=torch.int32)
    dk, dv, dt, ds, dd = on_gpu(kc, vc, table, src, dst)
    attn.kv_compact(dk, dv, dt, ds, dd)
    assert torch.equal(dk.cpu(), ref.compact(kc, table, src, dst))
    assert torch.equal(dv.cpu(), ref.compact(vc, table, src, dst))
    dd.fill_(-2)                                        # the first two destinations are outside
    kc, vc = dk.cpu(), dv.cpu()
    attn.kv_compact(dk, dv, dt, ds, dd)
    assert torch.equal(dk.cpu(), ref.compact(kc, table, src, dd.cpu()))


@gpu
@pytest.mark.parametrize("n", [1, 2, 63, 1000, 1024])
def test_compact_of_many_rows(n):
    gen = torch.Generator().manual_seed(n)
    kc, vc = torch.randn(2, 70, 16, 2, 64, generator=gen).half()
    table = torch.randperm(70, generator=gen)[:68].view(1, 68).to(torch.int32)
    src = torch.randperm(68 * 16, generator=gen)[:n].view(1, n).to(torch.int32)
    dst = torch.tensor([17], dtype=torch.int32)
    dk, dv, dt, ds, dd = on_gpu(kc, vc, table, src, dst)
    attn.kv_compact(dk, dv, dt, ds, dd)
    assert torch.equal(dk.cpu(), ref.compact(kc, table, src, dst))
    assert torch.equal(dv.cpu(), ref.compact(vc, table, src, dst))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 16), (1, 5, 3), (3, 37, 1), (2, 256, 64)])
def test_copy_pages_against_reference(dtype, hkv, d, bs):
    gen = torch.Generator().manual_seed(bs)
    kc, vc = torch.randn(2, 40, bs, hkv, d, generator=gen).to(dtype)
    perm = torch.randperm(40, generator=gen).to(torch.int32)
    src, dst = perm[:15].clone(), perm[20:35].clone()
    src[3:6] = src[0]                                   # one page forked often
    src[7], dst[9], src[11], dst[12] = -1, -5, 40, 2**31 - 1
    dk, dv, ds, dd = on_gpu(kc, vc, src, dst)
    attn.kv_copy_pages(dk, dv, ds, dd)
    assert torch.equal(dk.cpu(), ref.copy_pages(kc, src, dst))
    assert torch.equal(dv.cpu(), ref.copy_pages(vc, src, dst))


@gpu
def test_empty_calls_do_nothing():
    kc = torch.randn(4, 16, 2, 64, device=DEV)
    vc, keep = torch.randn_like(kc), kc.clone()
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    attn.kv_copy_pages(kc, vc, none, none)
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    attn.kv_compact(kc, vc, table, torch.zeros(2, 0, dtype=torch.int32, device=DEV),
                    torch.zeros(2, dtype=torch.int32, device=DEV))
    q = torch.zeros(0, 3, 4, 64, device=DEV)
    assert attn.gqa_tree_decode(q, kc, vc, table[:0], none).shape == q.shape
    cs = rope_table(4, 64).to(DEV)
    a, b = attn.qk_norm_rope(q, q[:, :, :2], None, None, cs, torch.zeros(0, 3, dtype=torch.int32, device=DEV))
    assert a.shape == q.shape and b.shape == (0, 3, 2, 64)
    assert torch.equal(kc, keep)


# --------------------------------------------------------------------------- a whole step
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_speculative_step_equals_decoding_the_accepted_tokens_one_by_one(dtype):
    """Fork, append a tree, attend, keep one path, compact: the cache and the attention of the path
    must be those of kv_append + gqa_decode of the same tokens, one at a time."""
    gen = torch.Generator().manual_seed(11)
    b, t, hq, hkv, d, bs, pages = 3, 7, 8, 2, 128, 16, 12
    lens = torch.tensor([130, 15, 64])                  # before the step
    kc, vc = torch.randn(2, b * pages + pages, bs, hkv, d, generator=gen).to(dtype).to(DEV)
    table = torch.arange(b * pages, dtype=torch.int32).view(b, pages).to(DEV)
    # sequence 2 continues on copies of its pages
    fresh = torch.arange(b * pages, b * pages + pages, dtype=torch.int32, device=DEV)
    attn.kv_copy_pages(kc, vc, table[2].contiguous(), fresh)
    table[2] = fresh
    parent = [-1, 0, 0, 1, 2, 4, -1]
    depth, bits = [], []
    for i, par in enumerate(parent):
        depth.append(0 if par < 0 else depth[par] + 1)
        bits.append((0 if par < 0 else bits[par]) | 1 << i)
    path = [0, 2, 4, 5]
    q = torch.randn(b, t, hq, d, generator=gen).to(dtype).to(DEV)
    k, v = torch.randn(2, b, t, hkv, d, generator=gen).to(dtype).to(DEV)
    w = (1 + 0.1 * torch.randn(2, d, generator=gen)).to(dtype).to(DEV)
    cs = rope_table(256, d).to(DEV)
    pos = (lens[:, None] + torch.tensor(depth)).to(torch.int32).to(DEV)
    slots = (lens[:, None] + torch.arange(t)).to(torch.int32).to(DEV)
    k1, v1 = kc.clone(), vc.clone()
    qr = attn.qk_norm_rope_append(q, k, v, w[0], w[1], cs, pos, kc, vc, table, slots=slots)
    total = (lens + t).to(torch.int32).to(DEV)
    mask = torch.tensor([bits] * b, device=DEV)
    out = attn.gqa_tree_decode(qr, kc, vc, table, total, mask)
    src = (lens[:, None] + torch.tensor(path)).to(torch.int32).to(DEV)
    attn.kv_compact(kc, vc, table, src, lens.to(torch.int32).to(DEV))
    for step, i in enumerate(path):
        at = (lens + step).to(torch.int32).to(DEV)
        q1, key = attn.qk_norm_rope(q[:, i].contiguous(), k[:, i].contiguous(), w[0], w[1], cs, at)
        assert torch.equal(q1, qr[:, i])
        attn.kv_append(key, v[:, i].contiguous(), k1, v1, table, at)
        one = attn.gqa_decode(q1, k1, v1, table, at + 1)
        # both within two roundings of the same value (fp32: the fp32 terms, below 1e-4)
        tol = max(4 * half_step(dtype), 1e-4) * float(vc.float().abs().max())
        assert (one.float() - out[:, i].float()).abs().max() <= tol
    for c, c1 in ((kc, k1), (vc, v1)):
        for s in range(b):
            n = int(lens[s]) + len(path)
            rows = torch.arange(n)
            page = table[s].cpu()[rows // bs].long()
            assert torch.equal(c[page, rows % bs], c1[page, rows % bs])


# --------------------------------------------------------------------------- refusals, without a GPU
def test_c_entry_points_refuse_bad_arguments():
    lib = _cabi.load()
    one = 1

    def tree(dtype=2, batch=2, tokens=4, hq=8, hkv=2, d=128, blocks=4, bs=16, pages=2, scale=0.1, kernel=0, q=one, ws=None):
        return lib.gqa_b200_tree_decode(q, one, one, one, one, None, None, one, dtype, batch, tokens, hq, hkv, d, blocks,
                                        bs, pages, scale, kernel, ws, 0, None)

    assert tree(dtype=5) == -2 and tree(batch=-1) == -8 and tree(tokens=0) == -15 and tree(tokens=65) == -15
    assert tree(hq=7) == -3 and tree(hkv=0) == -3 and tree(d=0) == -4 and tree(d=257) == -4
    assert tree(blocks=0) == -5 and tree(bs=0) == -5 and tree(pages=0) == -6
    assert tree(scale=0.0) == -7 and tree(scale=float("nan")) == -7 and tree(scale=float("inf")) == -7
    assert tree(kernel=2) == -11 and tree(q=None) == -1 and tree() == -9 and tree(blocks=2**31) == -13
    assert tree(batch=0) == 0
    ws = lib.gqa_b200_tree_workspace_bytes
    assert ws(2, 4, 8, 2, 128, 16, 64) > 0 and ws(2, 65, 8, 2, 128, 16, 64) == 0 and ws(0, 4, 8, 2, 128, 16, 64) == 0
    assert ws(64, 8, 32, 8, 128, 16, 256) % 256 == 0

    strides = (ctypes.c_int64 * 9)(*([128] * 9))

    def rope(dtype=2, wdtype=2, b=2, t=3, hq=8, hkv=2, d=128, rot=128, eps=1e-6, k_out=one, cache=None, st=strides, qw=one,
             kw=one, slots=one, maxpos=10):
        return lib.gqa_b200_qk_norm_rope(one, one, one, qw, kw, one, one, one, k_out, cache, cache, one, slots, dtype,
                                         wdtype, b, t, hq, hkv, d, rot, maxpos, st, eps, 0, 4, 16, 2, None)

    assert rope(dtype=4) == -2 and rope(wdtype=1) == -2 and rope(b=-1) == -8 and rope(hq=0) == -3 and rope(d=300) == -4
    assert rope(rot=3) == -16 and rope(rot=130) == -16 and rope(rot=-2) == -16 and rope(maxpos=2**31) == -16
    assert rope(eps=-1.0) == -7 and rope(eps=float("nan")) == -7
    assert rope(st=None) == -1 and rope(qw=None) == -1 and rope(k_out=None) == -1 and rope(cache=one, slots=None) == -1
    assert rope(b=0) == 0 and rope(t=0) == 0

    def compact(n=3, b=2, d=8, hkv=2, bs=4, pages=2, blocks=4, k=one):
        return lib.gqa_b200_kv_compact(k, one, one, one, one, 2, b, n, hkv, d, blocks, bs, pages, None)

    assert compact(n=1025) == -17 and compact(b=-1) == -8 and compact(n=-1) == -8 and compact(d=0) == -4
    assert compact(hkv=0) == -3 and compact(bs=0) == -5 and compact(pages=0) == -6 and compact(k=None) == -1
    assert compact(n=0) == 0 and compact(b=0) == 0

    def copy(n=3, d=8, hkv=2, bs=4, blocks=4, k=one):
        return lib.gqa_b200_kv_copy_pages(k, one, one, one, 2, n, hkv, d, blocks, bs, None)

    assert copy(n=-1) == -8 and copy(d=0) == -4 and copy(hkv=0) == -3 and copy(bs=0) == -5 and copy(k=None) == -1
    assert copy(n=0) == 0 and copy(blocks=2**31) == -13


def test_append_refuses_rows_that_lie_in_the_caches():
    """Another token's write could reach a row before it is read.  (Addresses only: nothing is launched.)"""
    lib = _cabi.load()
    b, t, hq, hkv, d, blocks, bs = 2, 3, 4, 2, 64, 5, 16
    cache = blocks * bs * hkv * d * 2
    kc, vc, rest = 1 << 20, (1 << 20) + 2 * cache, 1 << 30
    q_bytes, kv_bytes = b * t * hq * d * 2, b * t * hkv * d * 2

    def call(q=rest, k=rest + (1 << 20), v=rest + (2 << 20), st=None):
        st = st or [t * hq * d, hq * d, d] + [t * hkv * d, hkv * d, d] * 2
        out, meta = 1 << 40, 1 << 41
        return lib.gqa_b200_qk_norm_rope(q, k, v, None, None, meta, meta, out, None, kc, vc, meta, meta, 2, 2, b, t, hq, hkv,
                                         d, d, 10, (ctypes.c_int64 * 9)(*st), 1e-6, 0, blocks, bs, 4, None)

    for base in (kc, vc):
        assert call(q=base - q_bytes + 2) == -18 and call(q=base + cache - 2) == -18
        assert call(k=base) == -18 and call(k=base + cache - 128) == -18
        assert call(v=base - kv_bytes + 2) == -18 and call(v=base + cache // 2) == -18
    # rows before the address, by a negative stride; a token's rows far behind it
    assert call(k=kc + cache, st=[t * hq * d, hq * d, d, -t * hkv * d, hkv * d, d, t * hkv * d, hkv * d, d]) == -18
    assert call(v=kc - 4 * kv_bytes, st=[t * hq * d, hq * d, d, t * hkv * d, hkv * d, d, 2 * kv_bytes, hkv * d, d]) == -18
    assert "overlap" in _cabi.strerror(-18)


@gpu
def test_append_takes_rows_that_border_on_the_caches():
    """Queries, keys, values and both caches side by side in one allocation, and a key among the cache's rows refused."""
    b, t, hkv, d, pages, bs = 2, 3, 2, 64, 4, 16
    rows, cache = b * t * hkv * d, pages * bs * hkv * d
    gen = torch.Generator().manual_seed(0)
    flat = torch.randn(3 * rows + 2 * cache, generator=gen).half().to(DEV)
    q, kc, k, vc, v = (x.view(-1, bs, hkv, d) if x.numel() == cache else x.view(b, t, hkv, d)
                       for x in flat.split([rows, cache, rows, cache, rows]))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([[0, 17, 31], [5, 6, 7]], dtype=torch.int32, device=DEV)
    cs = rope_table(40, d).to(DEV)
    want_k, want_v = kc.cpu(), vc.cpu()
    with pytest.raises(RuntimeError, match="overlap"):
        attn.qk_norm_rope_append(q, kc.view(-1)[:rows].view(b, t, hkv, d), v, None, None, cs, pos, kc, vc, table)
    assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)
    keys = attn.qk_norm_rope(q, k, None, None, cs, pos)[1].cpu()
    attn.qk_norm_rope_append(q, k, v, None, None, cs, pos, kc, vc, table)
    live = torch.ones(b, t, dtype=torch.bool)
    ref.write_rows(want_k, keys, table.cpu(), pos.cpu(), live)
    ref.write_rows(want_v, v.cpu(), table.cpu(), pos.cpu(), live)
    assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)


def test_tree_refuses_a_workspace_that_meets_result_or_inputs():
    """(Addresses only: nothing is launched.)"""
    lib = _cabi.load()
    b, t, hq, hkv, d, blocks, bs, pages = 3, 4, 8, 2, 64, 40, 16, 12
    need = lib.gqa_b200_tree_workspace_bytes(b, t, hq, hkv, d, bs, pages)
    assert need > 4096
    size = dict(q=b * t * hq * d * 2, k=blocks * bs * hkv * d * 2, v=blocks * bs * hkv * d * 2, table=b * pages * 4, lens=b * 4,
                drafts=b * 4, mask=b * t * 8, out=b * t * hq * d * 2)
    at = {name: (i + 1) << 30 for i, name in enumerate(size)}
    names = ("q", "k", "v", "table", "lens", "drafts", "mask", "out")

    def call(ws, **change):
        a = {**at, **change}
        return lib.gqa_b200_tree_decode(*(a[n] for n in names), 2, b, t, hq, hkv, d, blocks, bs, pages, 0.1, 0, ws, need, None)

    for name in names:
        ws = (at[name] + size[name] - 1) // 256 * 256           # begins in the buffer's last bytes
        assert call(ws) == -18, name
        assert call(1 << 40, **{name: (1 << 40) + need - 1}) == -18, name
        assert call(1 << 40, **{name: (1 << 40) - size[name] + 1}) == -18, name
    for name in names[:-1]:
        assert call(1 << 40, out=at[name] + size[name] - 1) == -18, name


@gpu
def test_tree_workspace_may_border_on_result_and_inputs():
    case = tree_case([100, 17, 260], 4, 8, 2, 64, 16, torch.float16, seed=9)
    dq, dk, dv, dt, dl, dm, _ = on_gpu(*case)
    need = attn.tree_workspace_bytes(3, 4, 8, 2, 64, 16, dt.shape[1])
    flat = torch.empty(need + 2 * dq.nbytes, dtype=torch.uint8, device=DEV)
    assert dq.nbytes % 256 == 0
    q, ws, out = flat.split([dq.nbytes, need, dq.nbytes])
    q, out = q.view(dq.dtype).view(dq.shape), out.view(dq.dtype).view(dq.shape)
    q.copy_(dq)
    with pytest.raises(RuntimeError, match="overlap"):
        attn.gqa_tree_decode(q, dk, dv, dt, dl, dm, workspace=flat[: need])
    with pytest.raises(RuntimeError, match="overlap"):
        attn.gqa_tree_decode(q, dk, dv, dt, dl, dm, out=out, workspace=flat[2 * dq.nbytes:])
    check_tree(attn.gqa_tree_decode(q, dk, dv, dt, dl, dm, out=out, workspace=ws), case)
    assert torch.equal(q, dq)


def test_norm_rope_of_too_many_rows_has_a_status_of_its_own():
    """More groups of rows than a launch can number: the same status as the other sizes that exceed one."""
    lib = _cabi.load()

    def call(d, heads, batch=2**31 - 1, tokens=2):
        strides = (ctypes.c_int64 * 9)(*([0] * 9))
        return lib.gqa_b200_qk_norm_rope(16, 16, None, None, None, 16, 16, 16, 16, None, None, None, None, 2, 2, batch, tokens,
                                         heads, heads, d, d // 2 * 2, 10, strides, 1e-6, 0, 0, 0, 0, None)

    assert call(128, 1) == -13 and call(64, 4) == -13 and call(256, 8) == -13       # rows of whole chunks
    assert call(5, 4) == -13                                                        # the kernel for any row


def test_tree_workspace_of_too_many_rows_is_nothing():
    """tokens x q_heads beyond 2^20 is refused by the call: no scratch is asked for, and no int32 overflows on the way."""
    ws = _cabi.load().gqa_b200_tree_workspace_bytes
    assert ws(1, 64, 2**14, 2**14, 64, 16, 64) > 0
    for tokens, q_heads, kv_heads in [(64, 2**14 + 1, 1), (64, 2**30, 1), (33, 2**26, 1), (1, 2**20 + 1, 1), (64, 2**30, 2**30)]:
        assert ws(1, tokens, q_heads, kv_heads, 64, 16, 64) == 0


def test_front_doors_refuse_cpu_tensors():
    q = torch.zeros(2, 3, 4, 64)
    cache = torch.zeros(4, 16, 2, 64)
    i2 = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        attn.qk_norm_rope(q, q[:, :, :2], None, None, torch.zeros(4, 64), i2)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        attn.qk_norm_rope_append(q, q[:, :, :2], q[:, :, :2], None, None, torch.zeros(4, 64), i2, cache, cache, i2)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        attn.gqa_tree_decode(q, cache, cache, i2, i2[:, 0].contiguous())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        attn.kv_compact(cache, cache, i2, i2, i2[:, 0].contiguous())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        attn.kv_copy_pages(cache, cache, i2[0], i2[0])


@gpu
def test_front_doors_refuse_bad_tensors():
    q, k, v, table, lens, mask, _ = on_gpu(*tree_case([40, 30], 4, 8, 2, 64, 16, torch.float16))
    bad = [
        (dict(q=q[0]), r"\[B, T, Hq, D\]"), (dict(q=q.transpose(0, 1)), "contiguous"), (dict(q=q.float()), "dtype"),
        (dict(v=v[:1]), "v_cache shape"), (dict(table=table.long()), "int32"), (dict(lens=lens[:1]), "batch sizes"),
        (dict(mask=mask.int()), "tree_mask"), (dict(mask=mask[:, :2].contiguous()), "tree_mask"),
        (dict(q=q[:, :, :7].contiguous()), "divisible"), (dict(q=q[..., :32].contiguous()), "head_dim"),
        (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(drafts=lens.long()), "draft_lens"),
        (dict(q=q.repeat(1, 17, 1, 1), mask=None), r"\[1, 64\]"),
    ]
    for change, pattern in bad:
        a = dict(q=q, v=v, table=table, lens=lens, mask=mask, scale=None, drafts=None)
        a.update(change)
        with pytest.raises(RuntimeError, match=pattern):
            attn.gqa_tree_decode(a["q"], k, a["v"], a["table"], a["lens"], a["mask"], scale=a["scale"],
                                 draft_lens=a["drafts"])
    with pytest.raises(ValueError):
        attn.gqa_tree_decode(q, k, v, table, lens, mask, kernel="mma")
    with pytest.raises(RuntimeError, match="cannot run"):       # float32 has the CUDA-core kernel only
        attn.gqa_tree_decode(q.float(), k.float(), v.float(), table, lens, mask, kernel="tcgen05")

    cs = rope_table(16, 64).to(DEV)
    pos = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    w = torch.ones(64, dtype=torch.float16, device=DEV)
    kk = q[:, :, :2]
    rope_bad = [
        (dict(kw=None), "together"), (dict(qw=w[:32].contiguous()), r"\[D\]"), (dict(qw=w.bfloat16()), "float32 or"),
        (dict(cs=cs.half()), "float32"), (dict(cs=cs[:, :63].contiguous()), "even"), (dict(pos=pos.long()), "int32"),
        (dict(pos=pos[:, :2].contiguous()), "positions"), (dict(k=kk.float()), "dtype"), (dict(k=kk[:1]), "share batch"),
        (dict(q=q.transpose(2, 3)), "unit stride|share"), (dict(eps=-1.0), "eps"), (dict(q=q[:, 0], k=kk), "rank"),
        (dict(q_out=kk), "contiguous"),
    ]
    for change, pattern in rope_bad:
        a = dict(q=q, k=kk, qw=w, kw=w, cs=cs, pos=pos, eps=1e-6, q_out=None)
        a.update(change)
        with pytest.raises(RuntimeError, match=pattern):
            attn.qk_norm_rope(a["q"], a["k"], a["qw"], a["kw"], a["cs"], a["pos"], eps=a["eps"], q_out=a["q_out"])
    big = torch.empty(2 * q.numel(), dtype=q.dtype, device=DEV)
    shifted_in, shifted_out = big[: q.numel()].view(q.shape), big[64: 64 + q.numel()].view(q.shape)
    with pytest.raises(RuntimeError, match="overlap"):
        attn.qk_norm_rope(shifted_in, kk, w, w, cs, pos, q_out=shifted_out)

    for change, pattern in [(dict(v=v[:1]), "cache must"), (dict(v=v.float()), "share a dtype"),
                            (dict(src=pos.long()), "int32"), (dict(dst=lens[:1]), "metadata shape"),
                            (dict(src=torch.zeros(2, 1025, dtype=torch.int32, device=DEV)), "1024")]:
        a = dict(v=v, src=pos, dst=lens)
        a.update(change)
        with pytest.raises(RuntimeError, match=pattern):
            attn.kv_compact(k, a["v"], table, a["src"], a["dst"])
    with pytest.raises(RuntimeError, match="same length"):
        attn.kv_copy_pages(k, v, lens, lens[:1])
    with pytest.raises(RuntimeError, match="int32"):
        attn.kv_copy_pages(k, v, lens.long(), lens.long())


@gpu
def test_moves_refuse_caches_that_share_memory():
    """Both caches are moved by CTAs of their own: in shared memory one would read what the other has written."""
    both = torch.zeros(2 * 6 * 16 * 2 * 64, dtype=torch.float16, device=DEV)
    n = both.numel() // 2
    shape = (6, 16, 2, 64)
    k = both[:n].view(shape)
    table = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    src = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    dst = torch.zeros(2, dtype=torch.int32, device=DEV)
    rows = torch.zeros(2, 4, 2, 64, dtype=torch.float16, device=DEV)
    cs = rope_table(16, 64).to(DEV)
    for v in (k, both[64: 64 + n].view(shape)):
        with pytest.raises(RuntimeError, match="overlap"):
            attn.kv_compact(k, v, table, src, dst)
        with pytest.raises(RuntimeError, match="overlap"):
            attn.kv_copy_pages(k, v, dst, dst)
        with pytest.raises(RuntimeError, match="overlap"):
            attn.qk_norm_rope_append(rows, rows, rows, None, None, cs, src, k, v, table)
    attn.kv_copy_pages(k, both[n:].view(shape), dst, dst + 1)


@gpu
def test_norm_rope_in_place_refuses_a_tensor_that_is_queries_and_keys():
    """The heads of both are worked on side by side: rows that are still to be read would be overwritten."""
    x = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device=DEV)
    cs = rope_table(16, 64).to(DEV)
    pos = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    kc, vc = torch.zeros(2, 4, 16, 4, 64, dtype=torch.float16, device=DEV)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    for change in (dict(q_out=x), dict(k_out=x)):
        with pytest.raises(RuntimeError, match="overlap"):
            attn.qk_norm_rope(x, x, None, None, cs, pos, **change)
    for k, v in ((x, x.clone()), (x.clone(), x)):
        with pytest.raises(RuntimeError, match="overlap"):
            attn.qk_norm_rope_append(x, k, v, None, None, cs, pos, kc, vc, table, out=x)
    a, b = attn.qk_norm_rope(x, x, None, None, cs, pos)         # as two inputs it is as good as any other
    assert a.data_ptr() != b.data_ptr()


# --------------------------------------------------------------------------- paths that take more rows, pieces or tokens
def test_the_oracles_for_many_rows_are_the_oracles():
    case = tree_case([0, 1, 9, 40, 17], 6, 6, 2, 16, 4, torch.float32, seed=3, drafts=[6, 6, 0, 5, 99], masks="random")
    for masks in (case[5], None):
        args = (*case[:5], masks, case[6])
        for a, b in zip(ref.tree_decode(*args), ref.tree_decode_rows(*args)):
            torch.testing.assert_close(a, b, atol=1e-12, rtol=1e-12)
    gen = torch.Generator().manual_seed(0)
    x, w = torch.randn(2, 5, 3, 12, generator=gen), torch.randn(12, generator=gen)
    pos = torch.tensor([[0, 5, -1, 9, 3], [10, 2, 1, 1, 4]], dtype=torch.int32)
    for interleaved in (False, True):
        for weight in (w, None):
            args = (x, weight, rope_table(10, 8), pos)
            for a, b in zip(ref.norm_rope(*args, eps=1e-5, interleaved=interleaved),
                            ref.norm_rope_rows(*args, eps=1e-5, interleaved=interleaved)):
                torch.testing.assert_close(a, b, atol=1e-12, rtol=1e-12)


def check_tree_rows(got, case):
    """`check_tree` with the oracle for many rows."""
    q, k, v, table, lens, mask, dl = case
    want, mag = ref.tree_decode_rows(q, k, v, table, lens, mask, dl)
    d, dtype = q.shape[-1], q.dtype
    h = half_step(dtype)
    size = float(q.double().norm(dim=-1).max()) * float(k.double().norm(dim=-1).max()) / math.sqrt(d)
    fp32 = 2 * d * 2.0**-23 * size + 2.0**-20 + int(lens.max()) * 2.0**-23
    p_round = 0.0 if dtype == torch.float32 else h
    got = got.cpu().double()
    assert ((got - want).abs() <= h * want.abs() + (p_round + fp32) * mag + smallest(dtype)).all()
    for b in range(q.shape[0]):
        assert float((got[b] - want[b]).norm()) <= (h + fp32) * float(want[b].norm())


ROWS = [(8, 12), (16, 14), (40, 10), (60, 10)]          # drafted tokens, heads of two kv heads: 48, 112, 200, 300 rows each


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs", [16, 1, 24])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,hq", ROWS)
def test_tree_many_rows_and_hidden_infinities(dtype, t, hq, d, bs):
    """Several softmax warps, and two chains with a query tile each, look through the same drafted values."""
    lengths = [t, t + 20, 140, 256 + t // 2, 420]
    q, k, v, table, lens, _, _ = case = tree_case(lengths, t, hq, 2, d, bs, dtype, seed=t + d)
    shown = 0b1010 | 1 << (t - 2)
    mask = torch.full((len(lengths), t), shown if t < 64 else shown - (1 << 64), dtype=torch.int64)
    mask[0, 2] = 0                                              # no prefix either: nothing
    mask[2, t - 1] = 0                                          # the prefix alone
    clean = (q, k, v, table, lens, mask, None)
    bad = [float("nan"), float("inf"), float("-inf")]
    k, v = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        for j in range(t):
            if shown >> j & 1:
                continue
            page, line = int(table[b, (n - t + j) // bs]), (n - t + j) % bs
            k[page, line], v[page, line] = bad[j % 3], bad[(j + b) % 3]
        for pos in range(n, (n + bs - 1) // bs * bs):           # behind the end
            page = int(table[b, pos // bs])
            k[page, pos % bs], v[page, pos % bs] = bad[pos % 3], bad[(pos + 1) % 3]
    dq, dk, dv, dt, dl, dm, _ = on_gpu(q, k, v, table, lens, mask, None)
    got = attn.gqa_tree_decode(dq, dk, dv, dt, dl, dm)
    check_tree_rows(got, clean)
    assert torch.count_nonzero(got[0, 2]) == 0
    assert torch.equal(got, attn.gqa_tree_decode(dq, *on_gpu(clean[1], clean[2]), dt, dl, dm))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs", [16, 1, 24])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,hq", ROWS)
def test_tree_many_rows_and_infinities_that_some_see(dtype, t, hq, d, bs):
    """Drafted tokens on both sides of a tile's border, infinite in a column each of one kv head."""
    lengths = [t, 128 + t // 2, 256 + t - 2, 390]
    q, k, v, table, lens, mask, _ = tree_case(lengths, t, hq, 2, d, bs, dtype, seed=t * d)
    v = v.clone()
    want = torch.zeros(q.shape, dtype=torch.bool)
    for j, col in ((0, 3), (2, d - 1), (t // 2, d // 2 - 1), (t - 2, d // 2), (t - 1, 0)):
        seen = ((mask >> j) & 1) == 1
        want[:, :, hq // 2:, col] |= seen[:, :, None]
        for b, n in enumerate(lengths):
            v[int(table[b, (n - t + j) // bs]), (n - t + j) % bs, 1, col] = float("inf")
    got = attn.gqa_tree_decode(*on_gpu(q, k, v, table, lens, mask)).cpu()
    assert torch.equal(torch.isinf(got) & (got > 0), want)
    assert torch.isfinite(got[~want]).all()
    zero = v.clone()
    zero[torch.isinf(zero)] = 0                                 # what is finite must not have changed by it
    clean = attn.gqa_tree_decode(*on_gpu(q, k, zero, table, lens, mask)).cpu()
    assert torch.equal(got[~want], clean[~want])


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,hq,hkv,d", [(10, 20, 2, 256), (30, 20, 2, 256), (64, 8, 1, 200), (7, 80, 2, 256), (64, 64, 4, 128),
                                        (64, 32, 4, 64), (64, 32, 2, 80)])
def test_tree_wide_heads_and_several_blocks_of_rows(dtype, kernel, t, hq, hkv, d):
    """More rows than a query tile at D above 128, and more than two query tiles below."""
    case = tree_case([t, 200, 129, 700], t, hq, hkv, d, 16, dtype, seed=d + t, drafts=[t, t - 1, 0, t])
    dc = on_gpu(*case)
    check_tree_rows(attn.gqa_tree_decode(*dc[:6], draft_lens=dc[6], kernel=kernel), case)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,d,bs", [(400, 128, 16), (800, 64, 16), (250, 256, 16), (300, 128, 24), (1000, 37, 16)])
def test_tree_more_sequences_than_a_cta_has_threads(dtype, batch, d, bs):
    """The lengths are added up in several rounds."""
    gen = torch.Generator().manual_seed(batch)
    lengths = [int(x) for x in torch.randint(0, 150, (batch,), generator=gen)]
    lengths[0], lengths[-1], lengths[batch // 2] = 0, 0, 600
    case = tree_case(lengths, 3, 4, 2, d, bs, dtype, seed=batch)
    check_tree_rows(attn.gqa_tree_decode(*on_gpu(*case[:6])), case)


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 256), (torch.float32, 128),
                                     (torch.float32, 37), (torch.float16, 66)])
@pytest.mark.parametrize("t,hq,batch,tiles", [(1, 1, 1, 79), (3, 4, 1, 140), (2, 1, 2, 31), (2, 4, 2, 32), (2, 1, 2, 33), (5, 1, 2, 64),
                                              (2, 2, 2, 65)])
@pytest.mark.parametrize("trend", [6.0, -6.0])
def test_tree_sequences_cut_into_many_pieces(dtype, d, kernel, t, hq, batch, tiles, trend):
    """One kv head and a run a tile: the merge joins 32 pieces at a time and carries the rest on.  The scores rise
    (or fall) along the sequence, so that the maxima of the pieces differ and early (late) ones weigh little."""
    tile = 64 if kernel == "simt" or dtype == torch.float32 or d % 8 else 128
    lengths = [tiles * tile - 3, tiles * tile][:batch]
    q, k, v, table, lens, mask, _ = tree_case(lengths, t, hq, 1, d, 16, dtype, seed=tiles)
    q[..., 0] = 2.0
    for b, n in enumerate(lengths):
        pages = table[b, : (n + 15) // 16].long()
        ramp = torch.linspace(-0.5, 0.5, 16 * len(pages)).view(-1, 16, 1) * trend * math.sqrt(d) / 2
        k[pages, ..., 0] = ramp.to(dtype)
    case = (q, k, v, table, lens, mask, None)
    dc = on_gpu(*case[:6])
    got = attn.gqa_tree_decode(*dc, kernel=kernel)
    check_tree_rows(got, case)
    assert torch.equal(got, attn.gqa_tree_decode(*dc, kernel=kernel))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot,hq,hkv", [(64, 64, 7, 3), (128, 128, 6, 1), (80, 48, 8, 4), (256, 256, 7, 3), (96, 96, 5, 2),
                                          (128, 64, 9, 3)])
def test_norm_rope_of_many_tokens(dtype, interleaved, d, rot, hq, hkv):
    """Enough rows for four heads per group of lanes: heads that are no multiple of four, padding, slices of one
    projection's output, in place; the same bits as the same tokens in small calls, which take a head at a time."""
    gen = torch.Generator().manual_seed(d + hq)
    lanes = 8 if d <= 64 else 16 if d <= 128 else 32             # of a group
    b, heads = 2, hq + 2 * hkv
    t = 4 * 148 * 1024 // (b * (hq + hkv) * lanes) + 3           # a little more than four heads a group begin at
    qkv = torch.randn(b, t, heads, d, generator=gen).to(dtype)
    w = (1 + 0.2 * torch.randn(2, d, generator=gen)).to(dtype)
    cs = rope_table(300, rot)
    pos = torch.randint(0, 300, (b, t), generator=gen, dtype=torch.int32)
    pos[0, 5], pos[1, t - 1], pos[1, 0] = -1, 300, 2**31 - 1
    dqkv, dw, dcs, dp = on_gpu(qkv, w, cs, pos)
    q, k, v = dqkv.split([hq, hkv, hkv], 2)
    a, c = attn.qk_norm_rope(q, k, dw[0], dw[1], dcs, dp, interleaved=interleaved)
    for got, x, weight in ((a, qkv[:, :, :hq], w[0]), (c, qkv[:, :, hq:hq + hkv], w[1])):
        want, m = ref.norm_rope_rows(x, weight, cs, pos, eps=1e-6, interleaved=interleaved)
        assert ((got.cpu().double() - want).abs() <= half_step(dtype) * want.abs() + 2.1e-6 * m + smallest(dtype)).all()
    for lo in range(0, t, 97):
        part = slice(lo, min(t, lo + 97))
        x, y = attn.qk_norm_rope(q[:, part], k[:, part], dw[0], dw[1], dcs, dp[:, part].contiguous(), interleaved=interleaved)
        assert torch.equal(x, a[:, part]) and torch.equal(y, c[:, part])
    # into the cache: every other token's slot is out of range, one page is outside the pool
    bs, pages = 16, (t + 15) // 16
    kc, vc = torch.randn(2, b * pages, bs, hkv, d, generator=gen).to(dtype).to(DEV)
    want_k, want_v = kc.cpu(), vc.cpu()
    table = torch.randperm(b * pages, generator=gen).view(b, pages).to(torch.int32)
    table[1, 1] = -1
    slots = torch.arange(t, dtype=torch.int32).repeat(b, 1)
    slots[:, 1::2] = torch.tensor([[-1], [pages * bs]], dtype=torch.int32)
    out = attn.qk_norm_rope_append(q, k, v, dw[0], dw[1], dcs, dp, kc, vc, table.to(DEV), slots=slots.to(DEV),
                                   interleaved=interleaved)
    assert torch.equal(out, a)
    live = (pos >= 0) & (pos < 300)
    ref.write_rows(want_k, c.cpu(), table, slots, live)
    ref.write_rows(want_v, qkv[:, :, hq + hkv:], table, slots, live)
    assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)
    # in place, and without a norm
    q, k = q.contiguous(), k.contiguous()
    plain = attn.qk_norm_rope(q, k, None, None, dcs, dp, interleaved=interleaved)
    want, m = ref.norm_rope_rows(qkv[:, :, :hq], None, cs, pos, eps=1e-6, interleaved=interleaved)
    assert ((plain[0].cpu().double() - want).abs() <= half_step(dtype) * want.abs() + 2.1e-6 * m + smallest(dtype)).all()
    attn.qk_norm_rope(q, k, dw[0], dw[1], dcs, dp, interleaved=interleaved, q_out=q, k_out=k)
    assert torch.equal(q, a) and torch.equal(k, c)


@gpu
@pytest.mark.parametrize("kernel", ["auto", "simt"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bs", [16, 24])
def test_tree_lengths_outside_the_table_are_clamped(dtype, kernel, bs):
    """Negative lengths are empty sequences, longer ones than the table holds end with it, drafted tokens last."""
    q, k, v, table, lens, mask, _ = tree_case([240, 240, 240, 100], 5, 6, 2, 64, bs, dtype, seed=1)
    cap = table.shape[1] * bs
    wild = torch.tensor([2**31 - 1, -7, cap + 1, -2**31], dtype=torch.int32)
    case = (q, k, v, table, wild, mask, None)
    got = attn.gqa_tree_decode(*on_gpu(*case[:6]), kernel=kernel)
    check_tree_rows(got, (q, k, v, table, wild.clamp(0, cap), mask, None))
    assert torch.count_nonzero(got[1]) == 0 and torch.count_nonzero(got[3]) == 0
