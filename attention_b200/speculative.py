"""Front doors of the operators around a tree of drafted tokens on the paged cache.

One step of speculative decoding over the cache that ``gqa_decode`` reads:

    q = qk_norm_rope_append(q, k, v, ...)      # the drafted tokens into their pages
    out = gqa_tree_decode(q, ...)              # attention of the whole tree
    kv_compact(...)                            # the accepted path moved together
    kv_copy_pages(...)                         # pages of sequences that fork

``qk_norm_rope`` is the dense form of the first for ``gqa_prefill``.  The reference library has
none of these.  Same rules as the other operators: CUDA tensors of one device, the current
stream, no host read of device metadata, no synchronisation, no autograd, no CPU fallback.
"""

from __future__ import annotations

import ctypes
import math

import torch

from .core import _DTYPE_CODE, _check, _check_cuda_contiguous, _lib, _on_device, _raise_status, _stream_handle

_TREE_KERNEL_CODE = {"auto": 0, "simt": 1, "tcgen05": 4}
_tree_need: dict[tuple, int] = {}
_Strides = ctypes.c_int64 * 9


def _rows_4d(t, name, kv_like=None):
    """``[B,T,H,D]`` of a ``[B,T,H,D]`` or ``[B,H,D]`` tensor with unit stride in the last dimension."""
    _check(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _check(t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.dim() in (3, 4), f"{name} must be [B, T, H, D] or [B, H, D]")
    if t.dim() == 3:
        t = t.unsqueeze(1)
    _check(t.size(3) <= 1 or t.stride(3) == 1, f"{name} must have unit stride in its last dimension")
    return t


def _overlap(a, b) -> bool:
    """Whether the address ranges of two tensors (any strides) meet."""
    def span(t):
        if t.numel() == 0:
            return (0, 0)
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _check_rope(q, k, q_weight, k_weight, cos_sin, positions, eps):
    dims = q.dim()
    q4, k4 = _rows_4d(q, "q"), _rows_4d(k, "k")
    _check(k.dim() == dims, "q and k must have the same rank")
    _check(q4.shape[:2] == k4.shape[:2] and q4.size(3) == k4.size(3), "q/k must share batch, tokens and head_dim")
    _check(q4.size(2) > 0 and k4.size(2) > 0, "q/k must have heads")
    _check(0 < q4.size(3) <= 256, "supported head_dim is [1, 256]")
    _check(q.dtype == k.dtype, "q/k dtype must match")
    _check(q.dtype in _DTYPE_CODE, "q/k must be float32/float16/bfloat16")
    _check(k.device == q.device, "all tensors must use one CUDA device")
    _check((q_weight is None) == (k_weight is None), "q_weight and k_weight must be given together")
    if q_weight is not None:
        for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            _check_cuda_contiguous(t, name)
            _check(t.device == q.device, "all tensors must use one CUDA device")
            _check(t.dim() == 1 and t.size(0) == q4.size(3), f"{name} must be [D]")
            _check(t.dtype in (q.dtype, torch.float32), f"{name} must be float32 or of q's dtype")
        _check(q_weight.dtype == k_weight.dtype, "q_weight and k_weight dtype must match")
    _check_cuda_contiguous(cos_sin, "cos_sin")
    _check_cuda_contiguous(positions, "positions")
    _check(cos_sin.device == q.device and positions.device == q.device, "all tensors must use one CUDA device")
    _check(cos_sin.dim() == 2 and cos_sin.dtype == torch.float32, "cos_sin must be float32 [positions, rot_dim]")
    _check(cos_sin.size(1) % 2 == 0 and cos_sin.size(1) <= q4.size(3), "rot_dim must be even and at most head_dim")
    _check(positions.dtype == torch.int32, "positions must be int32")
    _check(positions.shape == q.shape[:dims - 2], "positions must be [B, T] ([B] for [B, H, D] inputs)")
    _check(math.isfinite(eps) and eps >= 0.0, "eps must be finite and not negative")
    _check(max(q4.shape) <= 2**31 - 1 and cos_sin.size(0) <= 2**31 - 1, "tensor sizes exceed int32 launch limits")
    return q4, k4


def _check_out(out, like, name, inputs):
    """A result buffer: contiguous, of `like`'s shape, and either `like` itself or apart from every input."""
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _check_cuda_contiguous(out, name)
    _check(out.shape == like.shape and out.dtype == like.dtype and out.device == like.device,
           f"{name} must have the shape, dtype and device of its input")
    same = out.data_ptr() == like.data_ptr() and like.is_contiguous()
    for t in inputs:
        if t is not None and not (same and t is like):
            _check(not _overlap(out, t), f"{name} must not overlap an input other than the one it replaces")
    return out


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _strides(*tensors):
    s = [x for t in tensors for x in t.stride()[:3]]
    return _Strides(*s, *([0] * (9 - len(s))))


def qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, *, eps=1e-6, interleaved=False, q_out=None,
                 k_out=None):
    """Per-head RMS norm of queries and keys and their position rotation, in one pass.

    ``q [B,T,Hq,D]``, ``k [B,T,Hkv,D]`` (or both without ``T``), float32/float16/bfloat16, any strides
    with unit stride in ``D`` (slices of a fused projection need no copy).  ``q_weight`` / ``k_weight``
    ``[D]`` scale the normalised rows, float32 or of ``q``'s dtype; both ``None`` leave the norm out.
    ``cos_sin`` float32 ``[positions, R]``: ``R/2`` cosines, then the ``R/2`` sines of each position's
    angles; the first ``R <= D`` elements are rotated, as pairs ``(i, i + R/2)`` or, ``interleaved``,
    ``(2i, 2i + 1)``.  ``positions`` int32 ``[B,T]`` (``[B]``); a token whose position is outside the
    table is padding and comes back as zeros.  Computed in fp32, rounded once.  Returns contiguous
    ``(q_out, k_out)``; a given ``q_out`` / ``k_out`` may be ``q`` / ``k`` itself.  No autograd support.
    """
    lib = _lib()
    eps = float(eps)
    q4, k4 = _check_rope(q, k, q_weight, k_weight, cos_sin, positions, eps)
    both = (q, k, q_weight, k_weight, cos_sin, positions)
    q_out = _check_out(q_out, q, "q_out", both)
    k_out = _check_out(k_out, k, "k_out", both)
    _check(not _overlap(q_out, k_out), "q_out and k_out must not overlap")
    if q4.size(0) == 0 or q4.size(1) == 0:
        return q_out, k_out
    with _on_device(q.device):
        rc = lib.gqa_b200_qk_norm_rope(
            q.data_ptr(), k.data_ptr(), None, _ptr(q_weight), _ptr(k_weight), cos_sin.data_ptr(),
            positions.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), None, None, None, None,
            _DTYPE_CODE[q.dtype], _DTYPE_CODE[q.dtype if q_weight is None else q_weight.dtype], q4.size(0),
            q4.size(1), q4.size(2), k4.size(2), q4.size(3), cos_sin.size(1), cos_sin.size(0), _strides(q4, k4), eps,
            int(interleaved), 0, 0, 0, _stream_handle(q.device))
    _raise_status(rc, "qk_norm_rope")
    return q_out, k_out


def qk_norm_rope_append(q, k, v, q_weight, k_weight, cos_sin, positions, k_cache, v_cache, block_table, *,
                        slots=None, eps=1e-6, interleaved=False, out=None):
    """``qk_norm_rope`` whose keys go straight into the paged cache, with ``v`` beside them.

    The row of token ``t`` of sequence ``b`` is written to position ``slots[b,t]`` (int32, default
    ``positions``) of its pages: page ``block_table[b, slot // block_size]``, row ``slot % block_size``.
    ``positions`` are the rotation's; the tokens of a tree share positions and differ in slots.  Nothing
    is written for padding (a position outside ``cos_sin``) or for a slot or page out of range; the
    caller owns distinct destinations.  Returns the rotated queries, shaped as ``q`` and contiguous;
    ``out`` may be ``q`` itself.  No autograd support.
    """
    lib = _lib()
    eps = float(eps)
    q4, k4 = _check_rope(q, k, q_weight, k_weight, cos_sin, positions, eps)
    v4 = _rows_4d(v, "v")
    if slots is None:
        slots = positions
    _check(v.shape == k.shape and v.dtype == k.dtype, "v must match k")
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache"), (block_table, "block_table"), (slots, "slots")):
        _check_cuda_contiguous(t, name)
    _check(all(t.device == q.device for t in (v, k_cache, v_cache, block_table, slots)),
           "all tensors must use one CUDA device")
    _check(k_cache.dim() == 4 and v_cache.shape == k_cache.shape, "cache must be [Nblocks, P, Hkv, D]")
    _check(k_cache.dtype == v_cache.dtype == q.dtype, "dtype mismatch")
    _check(k_cache.size(2) == k4.size(2) and k_cache.size(3) == k4.size(3), "cache head shape mismatch")
    _check(k_cache.size(0) > 0 and k_cache.size(1) > 0, "cache must have positive blocks and block_size")
    _check(max(k_cache.shape) <= 2**31 - 1, "tensor sizes exceed int32 launch limits")
    _check(block_table.dim() == 2 and block_table.size(0) == q4.size(0) and block_table.size(1) > 0
           and block_table.dtype == torch.int32, "block_table must be int32 [B, MaxPages]")
    _check(slots.dtype == torch.int32 and slots.shape == positions.shape, "slots must be int32 and shaped as positions")
    out = _check_out(out, q, "out", (q, k, v, q_weight, k_weight, cos_sin, positions, slots, k_cache, v_cache, block_table))
    if q4.size(0) == 0 or q4.size(1) == 0:
        return out
    with _on_device(q.device):
        rc = lib.gqa_b200_qk_norm_rope(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(q_weight), _ptr(k_weight), cos_sin.data_ptr(),
            positions.data_ptr(), out.data_ptr(), None, k_cache.data_ptr(), v_cache.data_ptr(),
            block_table.data_ptr(), slots.data_ptr(), _DTYPE_CODE[q.dtype],
            _DTYPE_CODE[q.dtype if q_weight is None else q_weight.dtype], q4.size(0), q4.size(1), q4.size(2),
            k4.size(2), q4.size(3), cos_sin.size(1), cos_sin.size(0), _strides(q4, k4, v4), eps, int(interleaved),
            k_cache.size(0), k_cache.size(1), block_table.size(1), _stream_handle(q.device))
    _raise_status(rc, "qk_norm_rope_append")
    return out


def tree_workspace_bytes(batch, tokens, q_heads, kv_heads, head_dim, block_size, max_pages) -> int:
    """Bytes of scratch ``gqa_tree_decode`` needs for this static shape."""
    return int(_lib().gqa_b200_tree_workspace_bytes(batch, tokens, q_heads, kv_heads, head_dim, block_size, max_pages))


def tree_tc_status(reset=True) -> int:
    """Status word of the tcgen05 tree kernel (synchronises): 0 ok, 2 = a bounded wait ran out."""
    return int(_lib().gqa_b200_tree_tc_status(1 if reset else 0))


def gqa_tree_decode(q, k_cache, v_cache, block_table, context_lens, tree_mask=None, *, draft_lens=None, scale=None,
                    out=None, workspace=None, kernel="auto"):
    """Paged GQA attention of up to 64 drafted tokens per sequence.

    ``q [B,T,Hq,D]``, caches, ``block_table`` and ``context_lens`` as for ``gqa_decode``; the lengths
    count the drafted tokens, which are the last ``draft_lens[b]`` (int32 ``[B]``, default ``T``) keys of
    a sequence.  Row ``i`` sees every earlier key and drafted token ``j`` iff bit ``j`` of
    ``tree_mask[b,i]`` (int64 ``[B,T]``, default the chain ``0 .. i``).  Rows that see nothing and rows
    from ``draft_lens[b]`` on come back as zeros; keys and values that a row does not see may hold
    anything.  ``workspace`` (uint8, at least ``tree_workspace_bytes(...)``, 256-byte aligned, contents
    irrelevant) is taken from the allocator for each call by default, so calls on different streams and
    captured graphs share nothing.  ``kernel``: ``"auto" | "simt" | "tcgen05"``.  No autograd support.
    """
    lib = _lib()
    for t, name in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache"), (block_table, "block_table"),
                    (context_lens, "context_lens")):
        _check_cuda_contiguous(t, name)
    _check(q.dim() == 4, "q must be [B, T, Hq, D]")
    _check(k_cache.dim() == 4, "k_cache must be [Nblocks, BlockSize, Hkv, D]")
    batch, tokens, q_heads, d = q.shape
    blocks, bs, kv_heads, kd = k_cache.shape
    dev = q.device
    scale = 1.0 / math.sqrt(d) if scale is None and d else float(scale or 0.0)
    _check(v_cache.shape == k_cache.shape, "v_cache shape mismatch")
    _check(block_table.dim() == 2, "block_table must be [B, MaxPages]")
    _check(context_lens.dim() == 1, "context_lens must be [B]")
    _check(k_cache.device == dev and v_cache.device == dev and block_table.device == dev
           and context_lens.device == dev, "all tensors must use one CUDA device")
    _check(q.dtype == k_cache.dtype == v_cache.dtype, "q/k/v dtype must match")
    _check(q.dtype in _DTYPE_CODE, "q/k/v must be float32/float16/bfloat16")
    _check(block_table.dtype == torch.int32 and context_lens.dtype == torch.int32,
           "block_table and context_lens must be int32")
    _check(batch == block_table.size(0) == context_lens.size(0), "batch sizes must match")
    _check(d == kd, "q head_dim and cache head_dim must match")
    _check(1 <= tokens <= 64, "drafted tokens per sequence must be in [1, 64]")
    _check(q_heads > 0 and kv_heads > 0 and q_heads % kv_heads == 0, "Hq must be divisible by Hkv")
    _check(0 < d <= 256, "supported head_dim is [1, 256]")
    _check(blocks > 0 and bs > 0, "cache must have positive blocks and block_size")
    _check(block_table.size(1) > 0, "block_table must have at least one page")
    _check(math.isfinite(scale) and scale > 0.0, "scale must be positive and finite")
    _check(max(batch, blocks, bs, block_table.size(1)) <= 2**31 - 1, "tensor sizes exceed int32 CUDA launch limits")
    if tree_mask is not None:
        _check_cuda_contiguous(tree_mask, "tree_mask")
        _check(tree_mask.dtype == torch.int64 and tree_mask.shape == (batch, tokens) and tree_mask.device == dev,
               "tree_mask must be int64 [B, T] on q's device")
    if draft_lens is not None:
        _check_cuda_contiguous(draft_lens, "draft_lens")
        _check(draft_lens.dtype == torch.int32 and draft_lens.shape == (batch,) and draft_lens.device == dev,
               "draft_lens must be int32 [B] on q's device")
    if kernel not in _TREE_KERNEL_CODE:
        raise ValueError("kernel must be auto, simt or tcgen05")
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_cuda_contiguous(out, "out")
        _check(out.shape == q.shape and out.dtype == q.dtype and out.device == dev, "out must match q")
        for t in (q, k_cache, v_cache, block_table, context_lens, tree_mask, draft_lens):
            _check(t is None or not _overlap(out, t), "out must not overlap an input")
    if batch == 0:
        return out
    with _on_device(dev):
        if workspace is None:
            key = (batch, tokens, q_heads, kv_heads, d, bs, block_table.size(1))
            need = _tree_need.get(key)
            if need is None:
                if len(_tree_need) >= 4096:
                    _tree_need.clear()
                need = _tree_need[key] = int(lib.gqa_b200_tree_workspace_bytes(*key))
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        else:
            _check(workspace.is_cuda and workspace.device == dev and workspace.is_contiguous()
                   and workspace.dtype == torch.uint8, "workspace must be a contiguous uint8 tensor on q's device")
        rc = lib.gqa_b200_tree_decode(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), context_lens.data_ptr(),
            _ptr(draft_lens), _ptr(tree_mask), out.data_ptr(), _DTYPE_CODE[q.dtype], batch, tokens, q_heads, kv_heads,
            d, blocks, bs, block_table.size(1), scale, _TREE_KERNEL_CODE[kernel], workspace.data_ptr(),
            workspace.numel(), _stream_handle(dev))
    _raise_status(rc, "gqa_tree_decode")
    return out


def _check_caches(k_cache, v_cache):
    _check_cuda_contiguous(k_cache, "k_cache")
    _check_cuda_contiguous(v_cache, "v_cache")
    _check(k_cache.dim() == 4 and v_cache.shape == k_cache.shape, "cache must be [Nblocks, P, Hkv, D]")
    _check(k_cache.dtype == v_cache.dtype and k_cache.dtype in _DTYPE_CODE,
           "caches must share a dtype of float32/float16/bfloat16")
    _check(v_cache.device == k_cache.device, "all tensors must share a device")
    _check(min(k_cache.shape) > 0, "invalid dimensions")
    _check(max(k_cache.shape) <= 2**31 - 1, "tensor sizes exceed int32 launch limits")


def kv_compact(k_cache, v_cache, block_table, src_positions, dst_positions):
    """Move K and V rows within sequences: position ``src_positions[b,i]`` to ``dst_positions[b] + i``.

    ``src_positions`` int32 ``[B,N]`` (``N <= 1024``), ``dst_positions`` int32 ``[B]``.  After a
    verification step the sources are the accepted tokens' positions and the destination the end of the
    prefix.  Within a sequence every row is read before any is written, so sources may repeat and be
    destinations too.  An entry whose source (``-1``: none) or destination is outside the table, or on a
    page outside the pool, is skipped.  A row that is written must not be used by another sequence of
    the call.
    """
    lib = _lib()
    _check_caches(k_cache, v_cache)
    for t, name in ((block_table, "block_table"), (src_positions, "src_positions"), (dst_positions, "dst_positions")):
        _check_cuda_contiguous(t, name)
        _check(t.device == k_cache.device, "all tensors must share a device")
        _check(t.dtype == torch.int32, "metadata must be int32")
    _check(block_table.dim() == 2 and src_positions.dim() == 2 and dst_positions.dim() == 1
           and block_table.size(0) == src_positions.size(0) == dst_positions.size(0) and block_table.size(1) > 0,
           "invalid metadata shape")
    _check(src_positions.size(1) <= 1024, "kv_compact moves at most 1024 rows per sequence")
    with _on_device(k_cache.device):
        rc = lib.gqa_b200_kv_compact(
            k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), src_positions.data_ptr(),
            dst_positions.data_ptr(), _DTYPE_CODE[k_cache.dtype], src_positions.size(0), src_positions.size(1),
            k_cache.size(2), k_cache.size(3), k_cache.size(0), k_cache.size(1), block_table.size(1),
            _stream_handle(k_cache.device))
    _raise_status(rc, "kv_compact")


def kv_copy_pages(k_cache, v_cache, src_pages, dst_pages):
    """Copy whole pages: K and V of page ``src_pages[i]`` to page ``dst_pages[i]`` (int32 ``[N]``).

    For sequences that fork (the last, partly filled page) or are moved.  A pair with an id outside the
    pool (``-1``: none) is skipped.  A source may occur often; the caller owns destinations that are
    distinct and not sources of the same call.
    """
    lib = _lib()
    _check_caches(k_cache, v_cache)
    for t, name in ((src_pages, "src_pages"), (dst_pages, "dst_pages")):
        _check_cuda_contiguous(t, name)
        _check(t.device == k_cache.device, "all tensors must share a device")
        _check(t.dtype == torch.int32 and t.dim() == 1, f"{name} must be int32 [N]")
    _check(src_pages.size(0) == dst_pages.size(0), "src_pages and dst_pages must have the same length")
    with _on_device(k_cache.device):
        rc = lib.gqa_b200_kv_copy_pages(
            k_cache.data_ptr(), v_cache.data_ptr(), src_pages.data_ptr(), dst_pages.data_ptr(),
            _DTYPE_CODE[k_cache.dtype], src_pages.size(0), k_cache.size(2), k_cache.size(3), k_cache.size(0),
            k_cache.size(1), _stream_handle(k_cache.device))
    _raise_status(rc, "kv_copy_pages")
