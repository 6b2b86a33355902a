"""Plain 64-bit restatements of the rotary embedding, the paged append and the
paged attention, and the inputs of their tests (CPU tensors).

Rounding bounds: a result rounded once to type t is off by at most
``half_step(t)`` relative to its value.
"""

import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def frequencies(rot, theta=10000.0, scaling=None, factor=1.0, trained_len=None):
    """float64 radians per position of each pair, and the amplitude."""
    i = torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1)
    if scaling == "ntk" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** -i
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        keep = ((trained_len * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    return f, 1.0


def rotate(x, positions, rot, interleaved, f, amplitude=1.0, inverse=False):
    """``x [..., T, H, D]`` in float64, rotated by ``positions [..., T]``; also |a| + |b| of each element's pair."""
    x = x.double()
    y, mag = x.clone(), torch.zeros_like(x)
    t = positions.double()[..., None, None] * f * (-1.0 if inverse else 1.0)
    c, s = torch.cos(t) * amplitude, torch.sin(t) * amplitude
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + (1 if interleaved else rot // 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * abs(amplitude)
    return y, mag


def rotate_bound(y, mag, dtype):
    """Bound on a rotation's error in ``dtype``: the one rounding, and in fp32 the
    angle (its distance to a quarter turn rounded to 24 bits: 2^-24 pi / 4), the
    polynomials (2^-24 each), the amplitude, two products and a sum (2^-24 each):
    below 2^-21 (|a| + |b|) together."""
    return half_step(dtype) * y.abs() + 2.0 ** -21 * mag


def paged_inputs(new, lens, H, D, page, dtype, g, spare=3, order="page"):
    """Pools with random pages handed out at random; every slot no key lies in, and every page no sequence has, holds
    NaN.  order: how the pools lie in memory ("page": [P, H, page, D], "slot": [P, page, H, D] permuted, "pair": k and
    v halves of one [P, 2, H, page, D])."""
    S = len(new)
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=g)
    width = max([1] + need) + 1
    table = torch.full((S, width), -1, dtype=torch.int32)
    if order == "slot":
        pools = [torch.full((total, page, H, D), math.nan, dtype=dtype).permute(0, 2, 1, 3) for _ in range(2)]
    elif order == "pair":
        both = torch.full((total, 2, H, page, D), math.nan, dtype=dtype)
        pools = [both[:, 0], both[:, 1]]
    else:
        pools = [torch.full((total, H, page, D), math.nan, dtype=dtype) for _ in range(2)]
    at = 0
    for s in range(S):
        table[s, :need[s]] = perm[at:at + need[s]].to(torch.int32)
        for j in range(need[s]):
            fill = min(page, lens[s] - j * page)
            for pool in pools:
                pool[perm[at + j], :, :fill] = torch.randn(H, fill, D, generator=g).to(dtype)
        at += need[s]
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    return pools[0], pools[1], table, cu, torch.tensor(lens, dtype=torch.int32)


def gather(pool, table, s, length, page):
    """Keys [0, length) of sequence s: ``[H, length, D]`` float64, and whether each has a page."""
    j = torch.arange(length)
    ids = table[s].long()[j // page]
    held = (ids >= 0) & (ids < pool.shape[0])
    rows = pool[ids.clamp(0, pool.shape[0] - 1), :, j % page].double()  # [length, H, D]
    rows[~held] = 0
    return rows.transpose(0, 1), held


def paged_attn(q, k_pages, v_pages, table, cu, lens, scale=None, window=None, selection=None):
    """float64 outputs and ``sum_j p_j |v_j|``, both ``[N, HQ, D]`` (zero rows for tokens of no sequence)."""
    N, HQ, D = q.shape
    H, page = k_pages.shape[1], k_pages.shape[2]
    G = HQ // H
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(N, HQ, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for s in range(len(lens)):
        lo, hi, length = int(cu[s]), int(cu[s + 1]), int(lens[s])
        if hi <= lo or length <= 0:
            continue
        k, held = gather(k_pages, table, s, length, page)
        v, _ = gather(v_pages, table, s, length, page)
        keys = torch.arange(length)
        pos = torch.arange(length - (hi - lo), length)
        seen = (keys <= pos[:, None]) & held
        if window is not None:
            seen &= keys >= pos[:, None] - window
        if selection is not None:
            seen &= selection[lo:hi, None]
        for h in range(HQ):
            x = (q[lo:hi, h].double() @ k[h // G].T) * scale
            x = x.masked_fill(~seen, -math.inf)
            m = x.amax(1, keepdim=True)
            m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
            p = torch.exp(x - m)
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total, torch.zeros_like(p))
            out[lo:hi, h] = p @ v[h // G]
            mag[lo:hi, h] = p @ v[h // G].abs()
    return out, mag


def attn_bound(out, mag, dtype):
    """The weights are rounded to ``dtype`` for the product with V (half_step of sum
    p |v|), the result once more; scores and sums in fp32: with |q| |k| scale up to
    about 12 at head dim 128, 128 2^-24 12 = 1e-4 of sum p |v| at most, taken twice
    for the exponential and the joining of pieces."""
    return half_step(dtype) * (mag + out.abs()) + 2e-4 * mag + 1e-30


def check(name, got, ref, bound):
    err = (got.detach().double().cpu() - ref).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} outside the bound, worst "
                                 f"{float((err / bound.clamp_min(1e-300))[bad].max()):.3g} times it; first at "
                                 f"{bad.nonzero()[0].tolist()}")
