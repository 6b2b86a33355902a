"""A key / value cache in pages and attention of new tokens over it
(``csrc/rotary.hip``, ``csrc/paged_attn.hip``).

A call works on the new tokens of several sequences, packed as everywhere in
this package: ``cu_seqlens [S + 1]`` bounds each sequence's tokens, and ``lens
[S]`` is its key count with those tokens included, so token i of sequence s has
position ``lens[s] - n_s + i``.  One call mixes single tokens with chunks of
prompts.  ``paged_append`` stores the tokens' keys (rotated on the way) and
values, ``paged_attn`` attends them to all keys of their sequence, with LoGo's
gate selection and local window as options.  Where ``ops.decode`` holds one
``[B, H, T, D]`` buffer a layer for sequences of one length bound, pages are
handed out as sequences grow and prompts may arrive in pieces.

Pages: ``k_pages`` and ``v_pages`` ``[P, H, page_size, D]`` (any strides that keep
rows dense and 16-byte aligned, so ``[P, page_size, H, D]`` may be passed as a
permuted view); ``block_table`` int32 ``[S, M]``, key j of sequence s in slot ``j %
page_size`` of page ``block_table[s, j // page_size]``.  Entries outside ``[0, P)``
name no page: nothing is stored to them, and attention does not see their keys.
"""

from typing import Optional

import torch

from .. import _lib
from .rotary import RotaryPlan

__all__ = ["paged_append", "paged_attn"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _check_cache(what, k_pages, v_pages, block_table, cu_seqlens, lens):
    """Refuses shapes and types that no call takes."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
        raise ValueError(f"{what}: k_pages and v_pages must be [P, H, page_size, D] of one shape and type")
    if k_pages.dtype not in _DTYPES:
        raise ValueError(f"{what} takes bf16 or fp16 pages, got {k_pages.dtype}")
    if block_table.dim() != 2 or cu_seqlens.dim() != 1 or lens.dim() != 1:
        raise ValueError(f"{what}: block_table must be [S, M], cu_seqlens [S + 1], lens [S]")
    if any(t.dtype != torch.int32 for t in (block_table, cu_seqlens, lens)):
        raise ValueError(f"{what}: block_table, cu_seqlens and lens must be int32")
    S = lens.shape[0]
    if block_table.shape[0] != S or cu_seqlens.shape[0] != S + 1:
        raise ValueError(f"{what}: block_table and cu_seqlens do not match {S} sequences")
    page, D = k_pages.shape[2:]
    if D not in (64, 128):
        raise ValueError(f"{what}: head dim {D} unsupported (64 or 128)")
    if page < 16 or page & (page - 1) or page > 65536:
        raise ValueError(f"{what}: page_size must be a power of two in [16, 65536], got {page}")
    for t in (k_pages, v_pages):
        if t.stride(3) != 1 or any(s % 8 for s in t.stride()[:3]) or t.stride(2) < D or t.data_ptr() % 16:
            raise ValueError(f"{what}: rows of the pages must be dense and 16-byte aligned")


def _guard(what, *tensors):
    """All tensors on one ROCm GPU."""
    _lib.require_gpu(*tensors)
    if any(t is not None and t.device != tensors[0].device for t in tensors):
        raise ValueError(f"{what}: tensors on different devices")


def _cache_arg(k_pages, v_pages, block_table, cu_seqlens, lens):
    """The ``logo_paged_cache`` of a call, and the tensors that have to live until its launch."""
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        block_table = block_table.contiguous()
    cu_seqlens, lens = cu_seqlens.contiguous(), lens.contiguous()
    c = _lib.PagedCacheArg()
    c.k, c.v = k_pages.data_ptr(), v_pages.data_ptr()
    c.k_page, c.k_head, c.k_slot, _ = k_pages.stride()
    c.v_page, c.v_head, c.v_slot, _ = v_pages.stride()
    c.pages, c.heads, c.page_size = k_pages.shape[:3]
    c.table, c.table_width = block_table.data_ptr(), block_table.shape[1]
    c.nseq = lens.shape[0]
    c.table_row = block_table.stride(0) if c.nseq > 1 else block_table.shape[1]
    c.cu, c.lens = cu_seqlens.data_ptr(), lens.data_ptr()
    return c, (block_table, cu_seqlens, lens)


def _rows16(x):
    """``x [N, H, D]`` with rows that 16-byte accesses reach (a copy where they do not)."""
    ok = x.stride(2) == 1 and x.data_ptr() % 16 == 0 and all(
        s % 8 == 0 or n <= 1 for s, n in zip(x.stride()[:2], x.shape[:2]))
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _strides(x):
    return tuple(s if n > 1 else 0 for s, n in zip(x.stride()[:2], x.shape[:2]))


def paged_append(k, v, k_pages, v_pages, block_table, cu_seqlens, lens, q=None, plan: Optional[RotaryPlan] = None):
    """Store the new tokens' keys ``k`` and values ``v`` (``[N, H, D]``, bf16 or
    fp16, any strides) in their pages, the keys rotated by their positions as
    ``plan`` says (None: as they are), and return ``q [N, HQ, D]`` rotated the same
    way as a new tensor (None without ``q``).  One launch, no gradients.

    Tokens behind the last sequence are not stored and have zero rows in the
    result, like tokens at negative positions; a token behind the block table or
    on an entry that names no page is not stored.  Two tokens of one call must not
    share a slot (sequences may share pages that the call does not write)."""
    _check_cache("paged_append", k_pages, v_pages, block_table, cu_seqlens, lens)
    if k.dim() != 3:
        raise ValueError("paged_append: k and v must be [N, H, D] of the pages' heads, head dim and type")
    N, H, D = k.shape
    if v.shape != k.shape or k.dtype != k_pages.dtype or v.dtype != k.dtype or k_pages.shape[1] != H \
            or k_pages.shape[3] != D:
        raise ValueError("paged_append: k and v must be [N, H, D] of the pages' heads, head dim and type")
    if q is not None and (q.dim() != 3 or q.shape[0] != N or q.shape[2] != D or q.dtype != k.dtype):
        raise ValueError("paged_append: q must be [N, HQ, D] of k's type")
    if plan is not None and plan.head_dim != D:
        raise ValueError(f"paged_append: the plan is for head dim {plan.head_dim}, not {D}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (k, v, q)):
        raise ValueError("paged_append has no gradients; call it under torch.no_grad()")
    _guard("paged_append", k_pages, v_pages, block_table, cu_seqlens, lens, k, v, q, plan.turns if plan else None)
    c, live = _cache_arg(k_pages, v_pages, block_table, cu_seqlens, lens)
    k, v = _rows16(k), _rows16(v)
    out = None
    if q is not None:
        q = _rows16(q)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if N == 0 or (q is not None and q.shape[1] == 0):
        return out
    if c.nseq == 0:
        return None if out is None else out.zero_()
    with _lib.on_device(k_pages):
        _lib.launch("logo_paged_append", _lib.lib().logo_paged_append, c, _lib.ptr(k), *_strides(k), _lib.ptr(v),
                    *_strides(v), _lib.ptr(q), *(_strides(q) if q is not None else (0, 0)), _lib.ptr(out),
                    q.shape[1] if q is not None else 0, N, D, _lib.ptr(plan.turns) if plan is not None else None,
                    plan.rot_dim if plan is not None else 0, int(plan is not None and plan.interleaved),
                    plan.amplitude if plan is not None else 1.0, _DTYPES[k.dtype], _lib.stream_of(k_pages))
    return out


def paged_attn(q, k_pages, v_pages, block_table, cu_seqlens, lens, max_q: Optional[int] = None,
               max_len: Optional[int] = None, scale: Optional[float] = None, window: Optional[int] = None,
               selection=None, out=None):
    """Attention of the new tokens ``q [N, HQ, D]`` over the cached keys of their
    own sequences (HQ a multiple of the pages' H; the new tokens' keys stored
    before, ``paged_append``): each token sees the keys up to its position and,
    with ``window``, none more than ``window`` before it (as ``swa_attn``).

    ``selection`` (bool ``[N]``): tokens with False read no key and get zero rows,
    as in ``sq_full_attn``.  ``max_q`` and ``max_len`` bound the new tokens and the
    keys of one sequence from the host (defaults: N and the block table's reach);
    they size the launch, and larger device values cost time only.  ``scale``
    defaults to ``D ** -0.5``.  Returns ``[N, HQ, D]``; rows behind the last sequence
    are zero, or left as they are in an ``out`` of the caller's (contiguous).  No
    gradients."""
    _check_cache("paged_attn", k_pages, v_pages, block_table, cu_seqlens, lens)
    if q.dim() != 3 or q.dtype != k_pages.dtype or q.shape[2] != k_pages.shape[-1]:
        raise ValueError("paged_attn: q must be [N, HQ, D] of the pages' head dim and type")
    N, HQ, D = q.shape
    H = k_pages.shape[1]
    if H == 0 or HQ % H:
        raise ValueError(f"paged_attn: {HQ} query heads are no multiple of the pages' {H}")
    if torch.is_grad_enabled() and q.requires_grad:
        raise ValueError("paged_attn has no gradients; call it under torch.no_grad()")
    if scale is None:
        scale = D ** -0.5
    if not (scale > 0 and scale < float("inf")):
        raise ValueError(f"paged_attn: scale must be positive and finite, got {scale}")
    if window is not None and window < 0:
        raise ValueError(f"paged_attn: window must be None or >= 0, got {window}")
    if selection is not None and (selection.dtype != torch.bool or selection.shape != (N,)):
        raise ValueError("paged_attn: selection must be bool [N]")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous()
                            or out.data_ptr() % 16):
        raise ValueError("paged_attn: out must be contiguous, of q's shape and type")
    _guard("paged_attn", k_pages, v_pages, block_table, cu_seqlens, lens, q, selection, out)
    c, live = _cache_arg(k_pages, v_pages, block_table, cu_seqlens, lens)
    selection = selection.contiguous() if selection is not None else None
    rest = out is None
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if N == 0 or HQ == 0:
        return out
    reach = c.table_width * c.page_size
    max_q = N if max_q is None else max(0, min(int(max_q), N))
    max_len = reach if max_len is None else max(0, min(int(max_len), reach))
    if window is None:
        window = -1
    window = min(int(window), (1 << 31) - 1)
    q = _rows16(q)
    lib = _lib.lib()
    nbytes = lib.logo_paged_attn_workspace_bytes(c.nseq, H, HQ, N, D, max_q, max_len, window,
                                                 selection is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    with _lib.on_device(k_pages):
        _lib.launch("logo_paged_attn", lib.logo_paged_attn, c, _lib.ptr(q), *_strides(q), _lib.ptr(out),
                    _lib.ptr(selection), HQ, N, D, max_q, max_len, float(scale), window, int(rest), _lib.ptr(ws), nbytes,
                    _DTYPES[q.dtype], _lib.stream_of(k_pages))
    return out
