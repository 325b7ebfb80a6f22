"""Serving from a paged key-value cache: writing it, attention over it, copying its pages — Python front ends.

One layer of a cache is a pair of tensors ``k_pages``, ``v_pages`` of shape ``[pages, kv_heads, page_size, head_dim]`` (views
with contiguous rows do).  Position ``j`` of sequence ``s`` lives in page ``table[s, j // page_size]`` at slot ``j % page_size``;
``lengths[s]`` counts the tokens of the sequence with its new ones.  The new tokens of all sequences are packed rows: those of
sequence ``s`` are rows ``offsets[s] .. offsets[s + 1]``, and they are its last tokens.  ``table``, ``lengths`` and ``offsets``
are int32 tensors that are read on the device: no call synchronises, and a captured one follows their contents.  Entries of
``table`` behind a sequence's last token are not read, and what slots behind it hold has no effect.  Rows outside every sequence, and sequences without
tokens, give zeros.

On CUDA the tensors are bf16 or fp16 with head_dim 64 or 128, else the call is refused; the CPU takes any float type.  An
entry of ``table`` that names no page, a length that the table cannot hold, or offsets that fall or lie outside the rows raise
on the CPU; on CUDA they are met on the device: the entry reads as zeros, is not written through, and
``ops.gemm.check_status`` raises.

Attention rounds each weight to the tensors' type before it multiplies a value, as the dense attention does; scores, weights'
sums and results are held in 32 bits until the end.  Against 64 bits its error is 1.2 to 1.4 times that of a form that is
rounded once (bf16 0.0023 in place of 0.0017 of the result's norm, fp16 0.00029 in place of 0.00021).

None of these operators has a backward pass: they refuse inputs that want a gradient, forward-mode tangents included.
:class:`incin_b200.cache.PagedCache` keeps the tables.
"""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _native as nat
from .gemm import status_word

c_void_p, c_int, c_ll, c_double = C.c_void_p, C.c_int, C.c_longlong, C.c_double

PAGE_SIZES = (16, 32, 64, 128)


# incin_paged_desc of the C header, field by field in native alignment.  Packed as bytes: a ctypes structure of as many fields
# takes three times as long to fill, which short calls notice.
_pack_desc = struct.Struct("@PP6qPqPP9ifPqqPPP").pack

nat.register_cuda_signatures({
    "incin_kv_append": (c_int, [c_void_p, c_double, c_void_p]),
    "incin_decode_attention_workspace": (c_ll, [c_void_p]),
    "incin_decode_attention": (c_int, [c_void_p, c_void_p]),
    "incin_prompt_attention_workspace": (c_ll, [c_void_p]),
    "incin_prompt_attention": (c_int, [c_void_p, c_void_p]),
    "incin_copy_pages": (c_int, [c_void_p] * 3 + [c_int, c_ll, c_int, c_ll, c_void_p, c_void_p]),
})

_KIND = {torch.bfloat16: nat.GEMM_IN_BF16, torch.float16: nat.GEMM_IN_FP16}


# ------------------------------------------------------------------------------------------------------------- checks
def _not_int_row(what: str, name: str, t):
    return ValueError(f"{what}: {name} must be int32 with contiguous rows, got {t.dtype}, strides {t.stride()}")


def check_kernels(what: str, dtype: torch.dtype, head_dim: int, group: int) -> None:
    """Raises where CUDA has no kernels for such a cache; ``group``: query heads of a key head."""
    if dtype not in _KIND or (head_dim != 64 and head_dim != 128):
        raise nat.NativeError(f"{what}: no kernel for {dtype} with head_dim {head_dim} (bf16 or fp16, head_dim 64 or 128)")
    if group > 128:
        raise nat.NativeError(f"{what}: {group} query heads share a key head (at most 128)")


def _no_gradient(what: str, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no backward pass and no forward-mode tangents either: call it with the primal tensors")


def _check(what: str, x, k_pages, v_pages, table, lengths, offsets, rows: int, n_heads: int):
    """The device's index (-1: the CPU does the call), what ``_launch`` wants to know of the shapes and the table's row stride,
    once everything about the arguments is in order.  These checks are a good part of a short call's time: no attribute is
    asked for twice."""
    shape, dtype = k_pages.shape, x.dtype
    if len(shape) != 4 or shape != v_pages.shape:
        raise ValueError(f"{what}: k_pages and v_pages must both be [pages, kv_heads, page_size, head_dim], got "
                         f"{tuple(shape)} and {tuple(v_pages.shape)}")
    pages, hkv, size, D = shape
    if size not in PAGE_SIZES:
        raise ValueError(f"{what}: page_size must be one of {PAGE_SIZES}, got {size}")
    if dtype is not k_pages.dtype or dtype is not v_pages.dtype or not dtype.is_floating_point:
        raise ValueError(f"{what}: rows and pages must have one float type, got {dtype}, {k_pages.dtype} and {v_pages.dtype}")
    if pages == 0 or hkv == 0 or n_heads <= 0 or n_heads % hkv:
        raise ValueError(f"{what}: {n_heads} query heads do not fall into {hkv} key heads ({pages} pages)")
    t_shape, l_shape = table.shape, lengths.shape
    if len(t_shape) != 2 or len(l_shape) != 1 or t_shape[0] != l_shape[0] or t_shape[0] == 0 or t_shape[1] == 0:
        raise ValueError(f"{what}: table must be [sequences, entries] and lengths [sequences], got {tuple(t_shape)} and "
                         f"{tuple(l_shape)}")
    seqs, width = t_shape
    t_row, t_one = table.stride()
    if table.dtype is not torch.int32 or (width > 1 and t_one != 1):
        raise _not_int_row(what, "table", table)
    if lengths.dtype is not torch.int32 or (seqs > 1 and lengths.stride(0) != 1):
        raise _not_int_row(what, "lengths", lengths)
    at = x.get_device()   # -1 on the CPU
    if k_pages.get_device() != at or v_pages.get_device() != at or table.get_device() != at or lengths.get_device() != at:
        raise ValueError(f"{what}: tensors on {[str(t.device) for t in (x, k_pages, v_pages, table, lengths)]}")
    if offsets is None:
        if rows != seqs:
            raise ValueError(f"{what}: {rows} rows for {seqs} sequences (one row each, or offsets)")
    else:
        if offsets.dim() != 1 or offsets.shape[0] != seqs + 1:
            raise ValueError(f"{what}: offsets must be [sequences + 1] = [{seqs + 1}], got {tuple(offsets.shape)}")
        if offsets.dtype is not torch.int32 or offsets.stride(0) != 1:
            raise _not_int_row(what, "offsets", offsets)
        if offsets.get_device() != at:
            raise ValueError(f"{what}: offsets on {offsets.device}, the others on {x.device}")
    if x.requires_grad or k_pages.requires_grad or v_pages.requires_grad or forward_ad._current_level >= 0:
        _no_gradient(what, x, k_pages, v_pages)
    kind = _KIND.get(dtype, -1)
    dims = (width, seqs, rows, pages, size, n_heads, hkv, D, kind)
    if at < 0:
        return at, dims, t_row
    check_kernels(what, dtype, D, n_heads // hkv)
    return at, dims, t_row


def _page_strides(what: str, name: str, t, at: int) -> tuple[int, int, int]:
    a, b, c, d = t.stride()
    if d != 1 or (a | b | c) % 8 or a <= 0 or b <= 0 or c <= 0 or at % 16:
        raise nat.NativeError(f"{what}: {name} needs contiguous rows that start on 16-byte boundaries, got strides {t.stride()}")
    return a, b, c


def _launch(fn, what: str, dims, t_row: int, x, x_at: int, x_row: int, x_head: int, k_pages, v_pages, table, lengths, offsets, out,
            scale: float = 0.0, args=(), workspace=None):
    k_at, v_at = k_pages.data_ptr(), v_pages.data_ptr()
    fields = (k_at, v_at, *_page_strides(what, "k_pages", k_pages, k_at), *_page_strides(what, "v_pages", v_pages, v_at), table.data_ptr(),
              t_row, lengths.data_ptr(), 0 if offsets is None else offsets.data_ptr(), *dims, scale, x_at, x_row, x_head, out.data_ptr())
    status = status_word(x.device).data_ptr()
    desc, room = _pack_desc(*fields, 0, status), None
    if workspace is not None:
        n = workspace(desc)
        if n:   # of this call alone: two captured graphs share none
            room = x.new_empty(n, dtype=torch.uint8)
            desc = _pack_desc(*fields, room.data_ptr(), status)
    nat.check(fn(desc, *args, nat.stream_ptr()), what)
    return out


# ------------------------------------------------------------------------------------------------------------- append
def kv_append(qkv, k_pages, v_pages, table, lengths, offsets=None, *, n_heads: int, theta: float | None = None):
    """Write the keys and values of new tokens into the cache and return their queries ``[rows, n_heads, head_dim]``.

    ``qkv``: packed projections ``[rows, (n_heads + 2 kv_heads) * head_dim]`` (query heads first, then key heads, then value
    heads).  With ``theta`` queries and keys are rotated to their positions first (rotate-half pairs, as
    :func:`~incin_b200.ops.functional.rope`).  ``offsets=None``: one new token per sequence; a sequence of length 0 is then an
    idle slot of the batch.  No two new tokens may share a slot."""
    if k_pages.dim() != 4 or qkv.dim() != 2:
        raise ValueError(f"kv_append: qkv must be [rows, width] and k_pages [pages, kv_heads, page_size, head_dim], got "
                         f"{tuple(qkv.shape)} and {tuple(k_pages.shape)}")
    (rows, wide), (_, hkv, _, D) = qkv.shape, k_pages.shape
    if wide != (n_heads + 2 * hkv) * D or D % 2:
        raise ValueError(f"kv_append: rows of {wide} elements, not ({n_heads} + 2 * {hkv}) heads of {D}")
    if theta is not None and not 1.0 <= theta < 1e300:
        raise ValueError(f"kv_append: theta must be at least 1, got {theta}")
    at, dims, t_row = _check("kv_append", qkv, k_pages, v_pages, table, lengths, offsets, rows, n_heads)
    if at < 0:
        return _append_cpu(qkv.unflatten(1, (n_heads + 2 * hkv, D)), k_pages, v_pages, table, lengths, offsets, n_heads, theta)
    if at != nat.device_index():
        with torch.cuda.device(qkv.device):
            return kv_append(qkv, k_pages, v_pages, table, lengths, offsets, n_heads=n_heads, theta=theta)
    q = qkv.new_empty((rows, n_heads, D))
    if rows == 0:
        return q
    (step, one), x_at = qkv.stride(), qkv.data_ptr()
    if one != 1 or step % 8 or step <= 0 or x_at % 16:   # the kernel wants dense heads on 16-byte boundaries
        qkv, step = qkv.clone(memory_format=torch.contiguous_format), wide
        x_at = qkv.data_ptr()
    _launch(nat.cuda().incin_kv_append, "kv_append", dims, t_row, qkv, x_at, step, D, k_pages, v_pages, table, lengths, offsets, q,
            args=(theta or 0.0,))
    increment_version((k_pages, v_pages))   # written in place, for autograd's knowledge
    return q


# ---------------------------------------------------------------------------------------------------------- attention
def decode_attention(q, k_pages, v_pages, table, lengths, *, scale: float | None = None):
    """Attention of one new token per sequence over all its cached tokens: ``q`` ``[sequences, heads, head_dim]`` -> the same
    shape.  Grouped heads as in :func:`~incin_b200.ops.functional.gqa_attention`; ``scale`` defaults to head_dim^-1/2."""
    return _attend("decode_attention", q, k_pages, v_pages, table, lengths, None, scale)


def prompt_attention(q, k_pages, v_pages, table, lengths, offsets, *, scale: float | None = None):
    """Causal attention of packed runs of new tokens over the cached tokens of their sequences: ``q``
    ``[rows, heads, head_dim]`` -> the same shape.  The new tokens' own keys and values are in the cache already
    (:func:`kv_append`); new token ``i`` of ``n`` sees the first ``lengths[s] - n + i + 1`` positions."""
    if offsets is None:
        raise ValueError("prompt_attention: offsets are required (decode_attention takes one row per sequence)")
    return _attend("prompt_attention", q, k_pages, v_pages, table, lengths, offsets, scale)


def _attend(what, q, k_pages, v_pages, table, lengths, offsets, scale):
    shape = q.shape
    if len(shape) != 3:
        raise ValueError(f"{what}: q must be [rows, heads, head_dim], got {tuple(shape)}")
    rows, n_heads, D = shape
    at, dims, t_row = _check(what, q, k_pages, v_pages, table, lengths, offsets, rows, n_heads)
    if D != dims[7]:
        raise ValueError(f"{what}: q must be [rows, heads, head_dim] of the cache's head_dim, got {tuple(shape)} and pages "
                         f"{tuple(k_pages.shape)}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 <= scale <= 1e38:
        raise ValueError(f"{what}: scale must lie in [0, 1e38], got {scale}")
    if at < 0:
        return _attend_cpu(q, k_pages, v_pages, table, lengths, offsets, scale)
    if at != nat.device_index():
        with torch.cuda.device(q.device):
            return _attend(what, q, k_pages, v_pages, table, lengths, offsets, scale)
    out = q.new_empty((rows, n_heads, D))
    if rows == 0:
        return out
    (a, b, one), x_at = q.stride(), q.data_ptr()
    if one != 1 or (a | b) % 8 or a <= 0 or b <= 0 or x_at % 16:   # the kernels want dense heads on 16-byte boundaries
        q, a, b = q.clone(memory_format=torch.contiguous_format), n_heads * D, D
        x_at = q.data_ptr()
    lib = nat.cuda()
    fn, room = ((lib.incin_decode_attention, lib.incin_decode_attention_workspace) if offsets is None else
                (lib.incin_prompt_attention, lib.incin_prompt_attention_workspace))
    return _launch(fn, what, dims, t_row, q, x_at, a, b, k_pages, v_pages, table, lengths, offsets, out, scale, workspace=room)


# -------------------------------------------------------------------------------------------------------------- pages
def copy_pages(storage, src, dst):
    """``storage[..., dst[i], :, :, :] = storage[..., src[i], :, :, :]`` for every pair ``i`` and all leading indices (layers,
    keys and values), in place; returns ``storage``.  ``storage``: dense ``[..., pages, kv_heads, page_size, head_dim]`` of any
    type whose pages are multiples of 16 bytes; ``src``, ``dst``: int32 ``[pairs]`` on its device.  A source may be named many
    times; a destination must be named once and be nobody's source (a page may be its own copy, and others' source then).
    Pairs that break this, or name no page, raise on the CPU; on CUDA they are left out and reported through
    ``ops.gemm.check_status``, the earliest of several equal destinations (of pairs that name pages) being kept."""
    shape, pairs, at = storage.shape, src.shape, storage.get_device()
    if len(shape) < 4 or not storage.is_contiguous():
        raise ValueError(f"copy_pages: storage must be dense [..., pages, kv_heads, page_size, head_dim], got {tuple(shape)}, "
                         f"strides {storage.stride()}")
    if len(pairs) != 1 or pairs != dst.shape or src.dtype is not torch.int32 or dst.dtype is not torch.int32:
        raise ValueError(f"copy_pages: src and dst must be int32 [pairs], got {tuple(src.shape)} {src.dtype} and {tuple(dst.shape)} {dst.dtype}")
    if src.get_device() != at or dst.get_device() != at:
        raise ValueError(f"copy_pages: tensors on {storage.device}, {src.device} and {dst.device}")
    if storage.requires_grad or forward_ad._current_level >= 0:
        _no_gradient("copy_pages", storage)
    *outer, pages, heads, size, D = shape
    page_bytes = heads * size * D * storage.element_size()
    outer = math.prod(outer)
    if page_bytes % 16:
        raise ValueError(f"copy_pages: pages of {page_bytes} bytes, not a multiple of 16")
    if at < 0:
        a, b = src.tolist(), dst.tolist()
        moves = [(i, j) for i, j in zip(a, b) if i != j]
        if any(not 0 <= i < pages for i in a + b):
            raise IndexError(f"copy_pages: page outside [0, {pages})")
        if len(set(b)) != len(b) or any(j in a for _, j in moves):
            raise IndexError("copy_pages: a destination is named twice or is also a source")
        if moves and storage.numel():
            flat = storage.view(outer, pages, -1)
            flat[:, [j for _, j in moves]] = flat[:, [i for i, _ in moves]]
        return storage
    n = pairs[0]
    if n == 0 or page_bytes * pages * outer == 0:
        return storage
    ptr = storage.data_ptr()
    if ptr % 16:
        raise nat.NativeError("copy_pages: storage must start on a 16-byte boundary")
    if at != nat.device_index():
        with torch.cuda.device(storage.device):
            return copy_pages(storage, src, dst)
    if n > 1:
        src, dst = src.contiguous(), dst.contiguous()
    nat.check(nat.cuda().incin_copy_pages(ptr, src.data_ptr(), dst.data_ptr(), n, outer, pages, page_bytes,
                                          status_word(storage.device).data_ptr(), nat.stream_ptr()), "copy_pages")
    increment_version(storage)
    return storage


# ----------------------------------------------------------------------------------------------------------- CPU twins
def _runs(k_pages, table, lengths, offsets, rows):
    """``(sequence, first row, new tokens, length)`` of every sequence, checked."""
    size = k_pages.shape[2]
    lens = lengths.tolist()
    offs = list(range(rows + 1)) if offsets is None else offsets.tolist()
    out = []
    for s, n in enumerate(lens):
        if not 0 <= n <= table.shape[1] * size:
            raise IndexError(f"sequence {s}: length {n}, its table holds {table.shape[1] * size}")
        used = table[s, :(n + size - 1) // size]
        if used.numel() and not 0 <= int(used.min()) <= int(used.max()) < k_pages.shape[0]:
            raise IndexError(f"sequence {s}: a page outside [0, {k_pages.shape[0]})")
        a, b = offs[s], offs[s + 1]
        if offsets is None and n == 0:
            b = a    # an idle slot
        if not 0 <= a <= b <= rows or b - a > n:
            raise IndexError(f"sequence {s}: rows {a}..{b} of {rows}, length {n}")
        out.append((s, a, b - a, n))
    return out


def _append_cpu(x, k_pages, v_pages, table, lengths, offsets, n_heads, theta):
    hkv, size, D = k_pages.shape[1:]
    q = torch.zeros(x.shape[0], n_heads, D, dtype=x.dtype, device=x.device)
    for s, at, n, total in _runs(k_pages, table, lengths, offsets, x.shape[0]):
        pos = torch.arange(total - n, total)
        rows = x[at:at + n]
        if theta is not None:
            angle = pos.double()[:, None] * theta ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)
            f = torch.promote_types(x.dtype, torch.float32)
            cs, sn = angle.cos().to(f)[:, None], angle.sin().to(f)[:, None]
            a, b = rows[:, :n_heads + hkv, :D // 2].to(f), rows[:, :n_heads + hkv, D // 2:].to(f)
            turned = torch.cat([a * cs - b * sn, b * cs + a * sn], -1).to(x.dtype)
            rows = torch.cat([turned, rows[:, n_heads + hkv:]], 1)
        q[at:at + n] = rows[:, :n_heads]
        page, slot = table[s].long()[pos // size], pos % size
        k_pages[page, :, slot] = rows[:, n_heads:n_heads + hkv]
        v_pages[page, :, slot] = rows[:, n_heads + hkv:]
    return q


def _attend_cpu(q, k_pages, v_pages, table, lengths, offsets, scale):
    hkv, size, D = k_pages.shape[1:]
    out = torch.zeros(q.shape, dtype=q.dtype)
    f = torch.promote_types(q.dtype, torch.float32)
    group = q.shape[1] // hkv
    for s, at, n, total in _runs(k_pages, table, lengths, offsets, q.shape[0]):
        pages = table[s, :(total + size - 1) // size].long()
        k, v = (t[pages].transpose(0, 1).reshape(hkv, -1, D)[:, :total].to(f).repeat_interleave(group, 0) for t in (k_pages, v_pages))
        z = torch.einsum("nhd,hkd->hnk", q[at:at + n].to(f), k) * scale
        for i in range(n):   # row by row, so that a key behind a row's last one does not enter it, not even as 0 * NaN
            seen = total - n + i + 1
            out[at + i] = torch.einsum("hk,hkd->hd", torch.softmax(z[:, i, :seen], -1), v[:, :seen]).to(q.dtype)
    return out
