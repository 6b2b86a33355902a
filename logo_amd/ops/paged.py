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

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .. import _torch_ops
from .rotary import RotaryPlan, rotary_plan

__all__ = ["paged_append", "paged_attn", "PagedStep", "PagedLogoCache"]


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
    share a slot (sequences may share pages that the call does not write), and no
    two rows of the pages the same memory."""
    _no_grad("paged_append", k, v, q, k_pages, v_pages)
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
    are zero, or left as they are in an ``out`` of the caller's (contiguous; q itself,
    or apart from all inputs).  No gradients."""
    _no_grad("paged_attn", q, k_pages, v_pages, out)
    if window is not None and window < 0:
        raise ValueError(f"paged_attn: window must be None or >= 0, got {window}")
    args = (q, k_pages, v_pages, block_table, cu_seqlens, lens, selection, -1 if max_q is None else max(0, max_q),
            -1 if max_len is None else max(0, max_len), q.shape[-1] ** -0.5 if scale is None else scale,
            -1 if window is None else window)
    if out is None:
        return _torch_ops.timed("logo_paged_attn", _torch_ops.ops().paged_attn, *args)
    _torch_ops.timed("logo_paged_attn", _torch_ops.ops().paged_attn_out, *args, out)
    return out


@dataclass(frozen=True)
class PagedStep:
    """One step of a server: the new tokens of some sequences, packed in the order
    of ``seqs``, as the operators take them.  ``table`` is the block table of the
    global branch, ``local_table`` that of the local one (pages behind the window
    are not in it), ``last`` the packed index of each sequence's last token."""

    seqs: Tuple[int, ...]
    new: Tuple[int, ...]
    cu: torch.Tensor
    lens: torch.Tensor
    last: torch.Tensor
    table: torch.Tensor
    local_table: torch.Tensor
    max_q: int
    max_len: int


class PagedLogoCache:
    """Paged key / value cache of a LoGo model: per layer a pool of pages for the
    global branch and one for the local branch, ``[P, H, page_size, D]`` each, and
    the pages of every sequence (host side).  The global pages of a sequence grow
    with it; of its local pages those behind the window go back to the pool.

    ``add()`` opens a sequence, ``step([(seq, tokens), ...])`` takes the pages that
    its next tokens need and returns the ``PagedStep`` to run, ``release(seq)`` gives
    its pages back.  Pools are filled on one stream; a page that was given back is
    handed out again to work that is queued behind."""

    def __init__(self, num_layers: int, kv_heads: int, head_dim: int, pages: int, local_pages: Optional[int] = None,
                 page_size: int = 64, window: int = 128, rope_theta: float = 10000.0, dtype=torch.bfloat16, device=None):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two of at least 16, got {page_size}")
        local_pages = pages if local_pages is None else local_pages
        self.page_size, self.window = page_size, window
        shape = lambda n: (n, kv_heads, page_size, head_dim)  # noqa: E731
        pool = lambda n: [torch.empty(shape(n), dtype=dtype, device=device) for _ in range(num_layers)]  # noqa: E731
        self.global_k, self.global_v = pool(pages), pool(pages)
        self.local_k, self.local_v = pool(local_pages), pool(local_pages)
        self.device = self.global_k[0].device if num_layers else torch.device(device or "cpu")
        self.rotary = rotary_plan(head_dim, theta=rope_theta, device=self.device)
        self._free, self._local_free = list(range(pages))[::-1], list(range(local_pages))[::-1]
        self._len: Dict[int, int] = {}
        self._pages: Dict[int, List[int]] = {}
        self._local: Dict[int, List[int]] = {}  # -1: given back
        self._next = 0

    def add(self) -> int:
        """Open a sequence without tokens."""
        seq = self._next
        self._next += 1
        self._len[seq], self._pages[seq], self._local[seq] = 0, [], []
        return seq

    def release(self, seq: int):
        """Give the sequence's pages back and forget it."""
        self._known(seq)
        self._free += self._pages.pop(seq)
        self._local_free += [p for p in self._local.pop(seq) if p >= 0]
        del self._len[seq]

    def length(self, seq: int) -> int:
        self._known(seq)
        return self._len[seq]

    def free_pages(self) -> Tuple[int, int]:
        """Pages left for the global and the local branch."""
        return len(self._free), len(self._local_free)

    def _known(self, seq):
        if seq not in self._len:
            raise ValueError(f"unknown sequence {seq}")

    def step(self, new: Sequence[Tuple[int, int]]) -> PagedStep:
        """Take the pages for ``new`` ((sequence, tokens) pairs, each sequence once)
        and return the step.  Raises RuntimeError, with nothing taken, if the pools
        do not hold them."""
        seqs, counts = tuple(int(s) for s, _ in new), tuple(int(n) for _, n in new)
        if not seqs or len(set(seqs)) != len(seqs):
            raise ValueError("a step takes each of its sequences once, and at least one")
        for s, n in zip(seqs, counts):
            self._known(s)
            if n < 1:
                raise ValueError(f"sequence {s}: a step takes at least one token, got {n}")
        size, lens = self.page_size, [self._len[s] + n for s, n in zip(seqs, counts)]
        need = [-(-n // size) for n in lens]
        # local pages that no token from here on sees
        gone = [max(0, self._len[s] - self.window) // size for s in seqs]
        back = sum(sum(p >= 0 for p in self._local[s][:g]) for s, g in zip(seqs, gone))
        take = sum(n - len(self._pages[s]) for s, n in zip(seqs, need))
        local_take = sum(n - max(len(self._local[s]), min(g, n)) for s, n, g in zip(seqs, need, gone))
        if take > len(self._free) or local_take > len(self._local_free) + back:
            raise RuntimeError(f"the cache is out of pages: {take} + {local_take} needed, {len(self._free)} + "
                               f"{len(self._local_free) + back} free")
        for s, g in zip(seqs, gone):
            local = self._local[s]
            for i in range(min(g, len(local))):
                if local[i] >= 0:
                    self._local_free.append(local[i])
                    local[i] = -1
        for s, n, g, length in zip(seqs, need, gone, lens):
            pages, local = self._pages[s], self._local[s]
            pages.extend(self._free.pop() for _ in range(n - len(pages)))
            local.extend([-1] * (min(g, n) - len(local)))
            local.extend(self._local_free.pop() for _ in range(n - len(local)))
            self._len[s] = length
        # one copy to the device: cu, lens, last, both tables
        S, width = len(seqs), max(need)
        buf = np.full(3 * S + 1 + 2 * S * width, -1, dtype=np.int32)
        cu = np.concatenate([[0], np.cumsum(counts)])
        buf[:S + 1], buf[S + 1:2 * S + 1], buf[2 * S + 1:3 * S + 1] = cu, lens, cu[1:] - 1
        tables = buf[3 * S + 1:].reshape(2, S, width)
        for i, s in enumerate(seqs):
            tables[0, i, :need[i]], tables[1, i, :need[i]] = self._pages[s], self._local[s]
        dev = torch.from_numpy(buf).to(self.device)
        tab = dev[3 * S + 1:].view(2, S, width)
        return PagedStep(seqs, counts, dev[:S + 1], dev[S + 1:2 * S + 1], dev[2 * S + 1:3 * S + 1], tab[0], tab[1],
                         max(counts), max(lens))
