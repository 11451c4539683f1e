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

import math
import struct

import torch

from .core import _DTYPE_CODE, _check, _check_cuda_contiguous, _lib, _on_device, _raise_status, _raw_stream, _stream_handle

_TREE_KERNEL_CODE = {"auto": 0, "simt": 1, "tcgen05": 4}
_I32 = torch.int32
_MAX = 2**31 - 1
_tree_need: dict[tuple, int] = {}
_pack_strides = struct.Struct("9q").pack
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _call(fn, device_index, device, *args):
    """``fn(*args, stream)`` with the tensors' device current; ``stream`` is its current one."""
    if _raw_stream is not None and _current_device() == device_index:
        return fn(*args, _raw_stream(device_index))
    with _on_device(device):
        return fn(*args, _stream_handle(device))


# Each front door first asks one boolean ("every check passes"), which costs a few microseconds of
# host time; only if that fails does the validator below it run, to raise the specific message.

def _span(t):
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a, b) -> bool:
    """Whether the address ranges of two tensors (any strides) meet."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _check_out(out, like, name, others):
    """A result buffer: contiguous, of the shape of the input `like`, and either `like` itself or apart from it; apart
    from the other inputs in any case (one of them may be the same tensor as `like`)."""
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _check_cuda_contiguous(out, name)
    _check(out.shape == like.shape and out.dtype == like.dtype and out.device == like.device,
           f"{name} must have the shape, dtype and device of its input")
    same = out.data_ptr() == like.data_ptr() and like.is_contiguous()
    _check((same or not _overlap(out, like)) and not any(t is not None and _overlap(out, t) for t in others),
           f"{name} must not overlap an input other than the one it replaces")
    return out


# --------------------------------------------------------------------------- norm and rotation
def _check_rows(t, name):
    _check(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _check(t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.dim() in (3, 4), f"{name} must be [B, T, H, D] or [B, H, D]")
    _check(t.size(-1) <= 1 or t.stride(-1) == 1, f"{name} must have unit stride in its last dimension")


def _validate_rope(q, k, q_weight, k_weight, cos_sin, positions, eps):
    _check_rows(q, "q")
    _check_rows(k, "k")
    dims = q.dim()
    _check(k.dim() == dims, "q and k must have the same rank")
    _check(q.shape[:dims - 2] == k.shape[:dims - 2] and q.size(-1) == k.size(-1), "q/k must share batch, tokens and head_dim")
    _check(q.size(-2) > 0 and k.size(-2) > 0, "q/k must have heads")
    _check(0 < q.size(-1) <= 256, "supported head_dim is [1, 256]")
    _check(q.dtype == k.dtype, "q/k dtype must match")
    _check(q.dtype in _DTYPE_CODE, "q/k must be float32/float16/bfloat16")
    _check(k.device == q.device, "all tensors must use one CUDA device")
    _check((q_weight is None) == (k_weight is None), "q_weight and k_weight must be given together")
    if q_weight is not None:
        for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            _check_cuda_contiguous(t, name)
            _check(t.device == q.device, "all tensors must use one CUDA device")
            _check(t.dim() == 1 and t.size(0) == q.size(-1), f"{name} must be [D]")
            _check(t.dtype in (q.dtype, torch.float32), f"{name} must be float32 or of q's dtype")
        _check(q_weight.dtype == k_weight.dtype, "q_weight and k_weight dtype must match")
    _check_cuda_contiguous(cos_sin, "cos_sin")
    _check_cuda_contiguous(positions, "positions")
    _check(cos_sin.device == q.device and positions.device == q.device, "all tensors must use one CUDA device")
    _check(cos_sin.dim() == 2 and cos_sin.dtype == torch.float32, "cos_sin must be float32 [positions, rot_dim]")
    _check(cos_sin.size(1) % 2 == 0 and cos_sin.size(1) <= q.size(-1), "rot_dim must be even and at most head_dim")
    _check(positions.dtype == _I32, "positions must be int32")
    _check(positions.shape == q.shape[:dims - 2], "positions must be [B, T] ([B] for [B, H, D] inputs)")
    _check(math.isfinite(eps) and eps >= 0.0, "eps must be finite and not negative")
    _check(max(q.shape) <= _MAX and cos_sin.size(0) <= _MAX, "tensor sizes exceed int32 launch limits")


def _rope_ok(dev, qs, ks, q, k, q_weight, k_weight, cos_sin, positions, eps) -> bool:
    try:
        dt = q.dtype
        d = qs[-1]
        rows, rot = cos_sin.shape
        if q_weight is not None:
            wt = q_weight.dtype
            if not ((wt == dt or wt == torch.float32) and k_weight.dtype == wt and q_weight.get_device() == dev
                    and k_weight.get_device() == dev and q_weight.shape == k_weight.shape == (d,)
                    and q_weight.is_contiguous() and k_weight.is_contiguous()):
                return False
        elif k_weight is not None:
            return False
        return (dev >= 0 and k.get_device() == dev and cos_sin.get_device() == dev and positions.get_device() == dev
                and 3 <= len(qs) <= 4 and len(ks) == len(qs) and qs[:-2] == ks[:-2] and ks[-1] == d and 0 < d <= 256
                and qs[-2] > 0 and ks[-2] > 0 and k.dtype == dt and dt in _DTYPE_CODE
                and (d == 1 or (q.stride(-1) == 1 and k.stride(-1) == 1))
                and cos_sin.dtype == torch.float32 and positions.dtype == _I32 and positions.shape == qs[:-2]
                and rot % 2 == 0 and rot <= d and cos_sin.is_contiguous() and positions.is_contiguous()
                and 0.0 <= eps < math.inf and max(qs) <= _MAX and rows <= _MAX)
    except (AttributeError, TypeError, ValueError):
        return False


def _strides3(t, four):
    s = t.stride()
    return s[:3] if four else (s[0], 0, s[1])


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
    ``(q_out, k_out)``; a given ``q_out`` / ``k_out`` may be ``q`` / ``k`` itself and must be apart from the
    other inputs.  No autograd support.
    """
    lib = _lib()
    eps = float(eps)
    try:
        dev, qs, ks = q.get_device(), q.shape, k.shape
    except AttributeError:
        dev, qs, ks = -1, (), ()
    if not _rope_ok(dev, qs, ks, q, k, q_weight, k_weight, cos_sin, positions, eps):
        _validate_rope(q, k, q_weight, k_weight, cos_sin, positions, eps)
        raise RuntimeError("invalid qk_norm_rope arguments")   # not reached: the line above raises
    if q_out is None and k_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        rest = (q_weight, k_weight, cos_sin, positions)
        q_out = _check_out(q_out, q, "q_out", (k, *rest))
        k_out = _check_out(k_out, k, "k_out", (q, *rest))
        _check(not _overlap(q_out, k_out), "q_out and k_out must not overlap")
    four = len(qs) == 4
    tokens = qs[1] if four else 1
    if qs[0] == 0 or tokens == 0:
        return q_out, k_out
    dt = _DTYPE_CODE[q.dtype]
    rc = _call(lib.gqa_b200_qk_norm_rope, dev, q.device,
               q.data_ptr(), k.data_ptr(), None, _ptr(q_weight), _ptr(k_weight), cos_sin.data_ptr(), positions.data_ptr(),
               q_out.data_ptr(), k_out.data_ptr(), None, None, None, None, dt,
               dt if q_weight is None else _DTYPE_CODE[q_weight.dtype], qs[0], tokens, qs[-2], ks[-2], qs[-1],
               cos_sin.size(1), cos_sin.size(0), _pack_strides(*_strides3(q, four), *_strides3(k, four), 0, 0, 0), eps,
               1 if interleaved else 0, 0, 0, 0)
    if rc:
        _raise_status(rc, "qk_norm_rope")
    return q_out, k_out


def _append_ok(dev, ks, k, v, k_cache, v_cache, block_table, slots, positions) -> bool:
    try:
        cs = k_cache.shape
        dt = k.dtype
        return (v.shape == ks and v.dtype == dt and (ks[-1] == 1 or v.stride(-1) == 1) and len(cs) == 4
                and v_cache.shape == cs and k_cache.dtype == dt and v_cache.dtype == dt and cs[2] == ks[-2]
                and cs[3] == ks[-1] and cs[0] > 0 and cs[1] > 0 and max(cs) <= _MAX and v.get_device() == dev
                and k_cache.get_device() == dev and v_cache.get_device() == dev and block_table.get_device() == dev
                and slots.get_device() == dev and k_cache.is_contiguous() and v_cache.is_contiguous()
                and block_table.is_contiguous() and slots.is_contiguous() and block_table.dim() == 2
                and block_table.size(0) == ks[0] and 0 < block_table.size(1) <= _MAX and block_table.dtype == _I32
                and slots.dtype == _I32 and slots.shape == positions.shape
                and abs(k_cache.data_ptr() - v_cache.data_ptr()) >= k_cache.nbytes)
    except (AttributeError, TypeError, ValueError):
        return False


def _validate_append(q, k, v, k_cache, v_cache, block_table, slots, positions):
    _check_rows(v, "v")
    _check(v.shape == k.shape and v.dtype == k.dtype, "v must match k")
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache"), (block_table, "block_table"), (slots, "slots")):
        _check_cuda_contiguous(t, name)
    _check(all(t.device == q.device for t in (v, k_cache, v_cache, block_table, slots)),
           "all tensors must use one CUDA device")
    _check(k_cache.dim() == 4 and v_cache.shape == k_cache.shape, "cache must be [Nblocks, P, Hkv, D]")
    _check(k_cache.dtype == v_cache.dtype == q.dtype, "dtype mismatch")
    _check(k_cache.size(2) == k.size(-2) and k_cache.size(3) == k.size(-1), "cache head shape mismatch")
    _check(k_cache.size(0) > 0 and k_cache.size(1) > 0, "cache must have positive blocks and block_size")
    _check(block_table.dim() == 2 and block_table.size(0) == q.size(0) and block_table.size(1) > 0
           and block_table.dtype == _I32, "block_table must be int32 [B, MaxPages]")
    _check(slots.dtype == _I32 and slots.shape == positions.shape, "slots must be int32 and shaped as positions")
    _check(max(*k_cache.shape, block_table.size(1)) <= _MAX, "tensor sizes exceed int32 launch limits")
    _check(not _overlap(k_cache, v_cache), "k_cache and v_cache must not overlap")


def qk_norm_rope_append(q, k, v, q_weight, k_weight, cos_sin, positions, k_cache, v_cache, block_table, *,
                        slots=None, eps=1e-6, interleaved=False, out=None):
    """``qk_norm_rope`` whose keys go straight into the paged cache, with ``v`` beside them.

    The row of token ``t`` of sequence ``b`` is written to position ``slots[b,t]`` (int32, default
    ``positions``) of its pages: page ``block_table[b, slot // block_size]``, row ``slot % block_size``.
    ``positions`` are the rotation's; the tokens of a tree share positions and differ in slots.  Nothing
    is written for padding (a position outside ``cos_sin``) or for a slot or page out of range; ``q``, ``k``
    and ``v`` must not overlap the caches, and the caller owns distinct destinations.  Returns the rotated queries, shaped as ``q`` and contiguous;
    ``out`` may be ``q`` itself.  No autograd support.
    """
    lib = _lib()
    eps = float(eps)
    if slots is None:
        slots = positions
    try:
        dev, qs, ks = q.get_device(), q.shape, k.shape
    except AttributeError:
        dev, qs, ks = -1, (), ()
    if not (_rope_ok(dev, qs, ks, q, k, q_weight, k_weight, cos_sin, positions, eps)
            and _append_ok(dev, ks, k, v, k_cache, v_cache, block_table, slots, positions)):
        _validate_rope(q, k, q_weight, k_weight, cos_sin, positions, eps)
        _validate_append(q, k, v, k_cache, v_cache, block_table, slots, positions)
        raise RuntimeError("invalid qk_norm_rope_append arguments")   # not reached: the lines above raise
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        out = _check_out(out, q, "out", (k, v, q_weight, k_weight, cos_sin, positions, slots, k_cache, v_cache,
                                         block_table))
    four = len(qs) == 4
    tokens = qs[1] if four else 1
    if qs[0] == 0 or tokens == 0:
        return out
    dt = _DTYPE_CODE[q.dtype]
    rc = _call(lib.gqa_b200_qk_norm_rope, dev, q.device,
               q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(q_weight), _ptr(k_weight), cos_sin.data_ptr(),
               positions.data_ptr(), out.data_ptr(), None, k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
               slots.data_ptr(), dt, dt if q_weight is None else _DTYPE_CODE[q_weight.dtype], qs[0], tokens, qs[-2],
               ks[-2], qs[-1], cos_sin.size(1), cos_sin.size(0),
               _pack_strides(*_strides3(q, four), *_strides3(k, four), *_strides3(v, four)), eps,
               1 if interleaved else 0, k_cache.size(0), k_cache.size(1), block_table.size(1))
    if rc:
        _raise_status(rc, "qk_norm_rope_append")
    return out


# --------------------------------------------------------------------------- tree attention
def tree_workspace_bytes(batch, tokens, q_heads, kv_heads, head_dim, block_size, max_pages) -> int:
    """Bytes of scratch ``gqa_tree_decode`` needs for this static shape."""
    return int(_lib().gqa_b200_tree_workspace_bytes(batch, tokens, q_heads, kv_heads, head_dim, block_size, max_pages))


def tree_tc_status(reset=True) -> int:
    """Status word of the tcgen05 tree kernel (synchronises): 0 ok, else a bounded wait ran out."""
    return int(_lib().gqa_b200_tree_tc_status(1 if reset else 0))


def _validate_tree(q, k_cache, v_cache, block_table, context_lens, tree_mask, draft_lens, scale):
    for t, name in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache"), (block_table, "block_table"),
                    (context_lens, "context_lens")):
        _check_cuda_contiguous(t, name)
    _check(q.dim() == 4, "q must be [B, T, Hq, D]")
    _check(k_cache.dim() == 4, "k_cache must be [Nblocks, BlockSize, Hkv, D]")
    dev = q.device
    _check(v_cache.shape == k_cache.shape, "v_cache shape mismatch")
    _check(block_table.dim() == 2, "block_table must be [B, MaxPages]")
    _check(context_lens.dim() == 1, "context_lens must be [B]")
    _check(k_cache.device == dev and v_cache.device == dev and block_table.device == dev
           and context_lens.device == dev, "all tensors must use one CUDA device")
    _check(q.dtype == k_cache.dtype == v_cache.dtype, "q/k/v dtype must match")
    _check(q.dtype in _DTYPE_CODE, "q/k/v must be float32/float16/bfloat16")
    _check(block_table.dtype == _I32 and context_lens.dtype == _I32, "block_table and context_lens must be int32")
    _check(q.size(0) == block_table.size(0) == context_lens.size(0), "batch sizes must match")
    _check(q.size(3) == k_cache.size(3), "q head_dim and cache head_dim must match")
    _check(1 <= q.size(1) <= 64, "drafted tokens per sequence must be in [1, 64]")
    _check(q.size(2) > 0 and k_cache.size(2) > 0 and q.size(2) % k_cache.size(2) == 0, "Hq must be divisible by Hkv")
    _check(0 < q.size(3) <= 256, "supported head_dim is [1, 256]")
    _check(k_cache.size(0) > 0 and k_cache.size(1) > 0, "cache must have positive blocks and block_size")
    _check(block_table.size(1) > 0, "block_table must have at least one page")
    _check(math.isfinite(scale) and scale > 0.0, "scale must be positive and finite")
    _check(max(*q.shape, *k_cache.shape, block_table.size(1)) <= _MAX, "tensor sizes exceed int32 CUDA launch limits")
    if tree_mask is not None:
        _check_cuda_contiguous(tree_mask, "tree_mask")
        _check(tree_mask.dtype == torch.int64 and tree_mask.shape == q.shape[:2] and tree_mask.device == dev,
               "tree_mask must be int64 [B, T] on q's device")
    if draft_lens is not None:
        _check_cuda_contiguous(draft_lens, "draft_lens")
        _check(draft_lens.dtype == _I32 and draft_lens.shape == q.shape[:1] and draft_lens.device == dev,
               "draft_lens must be int32 [B] on q's device")


def _tree_ok(dev, qs, ks, q, k_cache, v_cache, block_table, context_lens, tree_mask, draft_lens, scale) -> bool:
    try:
        dt = q.dtype
        batch, tokens, q_heads, d = qs
        blocks, bs, kv_heads, kd = ks
        rows, pages = block_table.shape
        if tree_mask is not None and not (tree_mask.dtype == torch.int64 and tree_mask.shape == qs[:2]
                                          and tree_mask.get_device() == dev and tree_mask.is_contiguous()):
            return False
        if draft_lens is not None and not (draft_lens.dtype == _I32 and draft_lens.shape == (batch,)
                                           and draft_lens.get_device() == dev and draft_lens.is_contiguous()):
            return False
        return (dev >= 0 and k_cache.get_device() == dev and v_cache.get_device() == dev
                and block_table.get_device() == dev and context_lens.get_device() == dev and v_cache.shape == ks
                and k_cache.dtype == dt and v_cache.dtype == dt and dt in _DTYPE_CODE and block_table.dtype == _I32
                and context_lens.dtype == _I32 and context_lens.shape == (batch,) and rows == batch and kd == d
                and 1 <= tokens <= 64 and q_heads > 0 and kv_heads > 0 and q_heads % kv_heads == 0 and 0 < d <= 256
                and blocks > 0 and bs > 0 and pages > 0 and 0.0 < scale < math.inf
                and q.is_contiguous() and k_cache.is_contiguous() and v_cache.is_contiguous()
                and block_table.is_contiguous() and context_lens.is_contiguous()
                and max(batch, q_heads, blocks, bs, pages) <= _MAX)
    except (AttributeError, TypeError, ValueError):
        return False


def gqa_tree_decode(q, k_cache, v_cache, block_table, context_lens, tree_mask=None, *, draft_lens=None, scale=None,
                    out=None, workspace=None, kernel="auto"):
    """Paged GQA attention of up to 64 drafted tokens per sequence.

    ``q [B,T,Hq,D]`` (``T * Hq <= 2**20``), caches, ``block_table`` and ``context_lens`` as for ``gqa_decode``; the lengths
    count the drafted tokens, which are the last ``draft_lens[b]`` (int32 ``[B]``, default ``T``) keys of
    a sequence.  Row ``i`` sees every earlier key and drafted token ``j`` iff bit ``j`` of
    ``tree_mask[b,i]`` (int64 ``[B,T]``, default the chain ``0 .. i``).  Rows that see nothing and rows
    from ``draft_lens[b]`` on come back as zeros; keys and values that a row does not see may hold
    anything.  ``workspace`` (uint8, at least ``tree_workspace_bytes(...)``, 256-byte aligned, contents
    irrelevant, apart from ``out`` and the inputs) is taken from the allocator for each call by default, so calls on different streams and
    captured graphs share nothing.  ``kernel``: ``"auto" | "simt" | "tcgen05"``.  No autograd support.
    """
    lib = _lib()
    try:
        dev, qs, ks = q.get_device(), q.shape, k_cache.shape
    except AttributeError:
        dev, qs, ks = -1, (), ()
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(qs[-1]) if qs and qs[-1] else 0.0
    if not _tree_ok(dev, qs, ks, q, k_cache, v_cache, block_table, context_lens, tree_mask, draft_lens, scale):
        _validate_tree(q, k_cache, v_cache, block_table, context_lens, tree_mask, draft_lens, scale)
        raise RuntimeError("invalid gqa_tree_decode arguments")   # not reached: the line above raises
    code = _TREE_KERNEL_CODE.get(kernel)
    if code is None:
        raise ValueError("kernel must be auto, simt or tcgen05")
    device = q.device
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_cuda_contiguous(out, "out")
        _check(out.shape == qs and out.dtype == q.dtype and out.device == device, "out must match q")
        for t in (q, k_cache, v_cache, block_table, context_lens, tree_mask, draft_lens):
            _check(t is None or not _overlap(out, t), "out must not overlap an input")
    batch, tokens, q_heads, d = qs
    blocks, bs, kv_heads, _ = ks
    if batch == 0:
        return out
    pages = block_table.size(1)
    if workspace is None:
        key = (batch, tokens, q_heads, kv_heads, d, bs, pages)
        need = _tree_need.get(key)
        if need is None:
            if len(_tree_need) >= 4096:
                _tree_need.clear()
            need = _tree_need[key] = int(lib.gqa_b200_tree_workspace_bytes(*key))
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    else:
        _check(workspace.is_cuda and workspace.device == device and workspace.is_contiguous()
               and workspace.dtype == torch.uint8, "workspace must be a contiguous uint8 tensor on q's device")
        need = workspace.numel()
    rc = _call(lib.gqa_b200_tree_decode, dev, device,
               q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), context_lens.data_ptr(),
               _ptr(draft_lens), _ptr(tree_mask), out.data_ptr(), _DTYPE_CODE[q.dtype], batch, tokens, q_heads, kv_heads,
               d, blocks, bs, pages, scale, code, workspace.data_ptr(), need)
    if rc:
        _raise_status(rc, "gqa_tree_decode")
    return out


# --------------------------------------------------------------------------- moves in the cache
def _caches_ok(dev, cs, k_cache, v_cache) -> bool:
    return (dev >= 0 and v_cache.get_device() == dev and len(cs) == 4 and v_cache.shape == cs and k_cache.dtype in _DTYPE_CODE
            and v_cache.dtype == k_cache.dtype and k_cache.is_contiguous() and v_cache.is_contiguous() and min(cs) > 0
            and max(cs) <= _MAX and abs(k_cache.data_ptr() - v_cache.data_ptr()) >= k_cache.nbytes)


def _validate_caches(k_cache, v_cache):
    _check_cuda_contiguous(k_cache, "k_cache")
    _check_cuda_contiguous(v_cache, "v_cache")
    _check(k_cache.dim() == 4 and v_cache.shape == k_cache.shape, "cache must be [Nblocks, P, Hkv, D]")
    _check(k_cache.dtype == v_cache.dtype and k_cache.dtype in _DTYPE_CODE,
           "caches must share a dtype of float32/float16/bfloat16")
    _check(v_cache.device == k_cache.device, "all tensors must share a device")
    _check(min(k_cache.shape) > 0, "invalid dimensions")
    _check(max(k_cache.shape) <= _MAX, "tensor sizes exceed int32 launch limits")
    _check(not _overlap(k_cache, v_cache), "k_cache and v_cache must not overlap")


def _compact_ok(dev, cs, k_cache, v_cache, block_table, src_positions, dst_positions) -> bool:
    try:
        rows, pages = block_table.shape
        b, n = src_positions.shape
        return (_caches_ok(dev, cs, k_cache, v_cache) and block_table.get_device() == dev and src_positions.get_device() == dev
                and dst_positions.get_device() == dev and block_table.dtype == _I32 and src_positions.dtype == _I32
                and dst_positions.dtype == _I32 and block_table.is_contiguous() and src_positions.is_contiguous()
                and dst_positions.is_contiguous() and rows == b and dst_positions.shape == (b,) and 0 < pages <= _MAX
                and n <= 1024)
    except (AttributeError, TypeError, ValueError):
        return False


def _validate_compact(k_cache, v_cache, block_table, src_positions, dst_positions):
    _validate_caches(k_cache, v_cache)
    for t, name in ((block_table, "block_table"), (src_positions, "src_positions"), (dst_positions, "dst_positions")):
        _check_cuda_contiguous(t, name)
        _check(t.device == k_cache.device, "all tensors must share a device")
        _check(t.dtype == _I32, "metadata must be int32")
    _check(block_table.dim() == 2 and src_positions.dim() == 2 and dst_positions.dim() == 1
           and block_table.size(0) == src_positions.size(0) == dst_positions.size(0) and block_table.size(1) > 0,
           "invalid metadata shape")
    _check(src_positions.size(1) <= 1024, "kv_compact moves at most 1024 rows per sequence")


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
    try:
        dev, cs = k_cache.get_device(), k_cache.shape
    except AttributeError:
        dev, cs = -1, ()
    if not _compact_ok(dev, cs, k_cache, v_cache, block_table, src_positions, dst_positions):
        _validate_compact(k_cache, v_cache, block_table, src_positions, dst_positions)
        raise RuntimeError("invalid kv_compact arguments")   # not reached: the line above raises
    rc = _call(lib.gqa_b200_kv_compact, dev, k_cache.device,
               k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), src_positions.data_ptr(),
               dst_positions.data_ptr(), _DTYPE_CODE[k_cache.dtype], src_positions.size(0), src_positions.size(1), cs[2],
               cs[3], cs[0], cs[1], block_table.size(1))
    if rc:
        _raise_status(rc, "kv_compact")


def _copy_ok(dev, cs, k_cache, v_cache, src_pages, dst_pages) -> bool:
    try:
        return (_caches_ok(dev, cs, k_cache, v_cache) and src_pages.get_device() == dev and dst_pages.get_device() == dev
                and src_pages.dtype == _I32 and dst_pages.dtype == _I32 and src_pages.dim() == 1
                and src_pages.shape == dst_pages.shape and src_pages.is_contiguous() and dst_pages.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        return False


def _validate_copy(k_cache, v_cache, src_pages, dst_pages):
    _validate_caches(k_cache, v_cache)
    for t, name in ((src_pages, "src_pages"), (dst_pages, "dst_pages")):
        _check_cuda_contiguous(t, name)
        _check(t.device == k_cache.device, "all tensors must share a device")
        _check(t.dtype == _I32 and t.dim() == 1, f"{name} must be int32 [N]")
    _check(src_pages.size(0) == dst_pages.size(0), "src_pages and dst_pages must have the same length")


def kv_copy_pages(k_cache, v_cache, src_pages, dst_pages):
    """Copy whole pages: K and V of page ``src_pages[i]`` to page ``dst_pages[i]`` (int32 ``[N]``).

    For sequences that fork (the last, partly filled page) or are moved.  A pair with an id outside the
    pool (``-1``: none) is skipped.  A source may occur often; the caller owns destinations that are
    distinct and not sources of the same call.
    """
    lib = _lib()
    try:
        dev, cs = k_cache.get_device(), k_cache.shape
    except AttributeError:
        dev, cs = -1, ()
    if not _copy_ok(dev, cs, k_cache, v_cache, src_pages, dst_pages):
        _validate_copy(k_cache, v_cache, src_pages, dst_pages)
        raise RuntimeError("invalid kv_copy_pages arguments")   # not reached: the line above raises
    rc = _call(lib.gqa_b200_kv_copy_pages, dev, k_cache.device,
               k_cache.data_ptr(), v_cache.data_ptr(), src_pages.data_ptr(), dst_pages.data_ptr(),
               _DTYPE_CODE[k_cache.dtype], src_pages.size(0), cs[2], cs[3], cs[0], cs[1])
    if rc:
        _raise_status(rc, "kv_copy_pages")
