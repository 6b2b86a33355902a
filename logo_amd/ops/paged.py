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

from .. import _torch_ops
from .rotary import RotaryPlan

__all__ = ["paged_append", "paged_attn"]


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradients; call it under torch.no_grad()")


def paged_append(k, v, k_pages, v_pages, block_table, cu_seqlens, lens, q=None, plan: Optional[RotaryPlan] = None):
    """Store the new tokens' keys ``k`` and values ``v`` (``[N, H, D]``, bf16 or
    fp16, any strides) in their pages, the keys rotated by their positions as
    ``plan`` says (None: as they are), and return ``q [N, HQ, D]`` rotated the same
    way as a new tensor (None without ``q``).  One launch, no gradients.

    Tokens behind the last sequence are not stored and have zero rows in the
    result, like tokens at negative positions; a token behind the block table or
    on an entry that names no page is not stored.  Two tokens of one call must not
    share a slot (sequences may share pages that the call does not write)."""
    _no_grad("paged_append", k, v, q)
    rot = (None, 0, 0, False, 1.0) if plan is None else (plan.turns, plan.head_dim, plan.rot_dim, plan.interleaved,
                                                         plan.amplitude)
    out = _torch_ops.timed("logo_paged_append", _torch_ops.ops().paged_append, k, v, k_pages, v_pages, block_table,
                           cu_seqlens, lens, q, *rot)
    return None if q is None else out


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
    they choose the kernel, and larger device values cost time only.  ``scale``
    defaults to ``D ** -0.5``.  Returns ``[N, HQ, D]``; rows behind the last sequence
    are zero, or left as they are in an ``out`` of the caller's (contiguous).  No
    gradients."""
    _no_grad("paged_attn", q)
    if window is not None and window < 0:
        raise ValueError(f"paged_attn: window must be None or >= 0, got {window}")
    args = (q, k_pages, v_pages, block_table, cu_seqlens, lens, selection, -1 if max_q is None else max(0, max_q),
            -1 if max_len is None else max(0, max_len), q.shape[-1] ** -0.5 if scale is None else scale,
            -1 if window is None else window)
    if out is None:
        return _torch_ops.timed("logo_paged_attn", _torch_ops.ops().paged_attn, *args)
    _torch_ops.timed("logo_paged_attn", _torch_ops.ops().paged_attn_out, *args, out)
    return out
