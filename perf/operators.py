"""Speed cases of the rotary embedding by positions, of the append to a paged
key / value cache with that rotation on the way, and of attention of new tokens
over such a cache.

``listed`` names the cases, ``draw`` gives further ones of the same ranges,
``prepare`` makes a case's inputs on the GPU from a seed, ``run`` is one pass:
in plain torch operations where ``own`` is false, through this package's
operators where it is true.  ``exact`` is the same result in 64 bits and
``work`` what a pass cannot do without.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TRAINED_LEN = 8192  # positions that a frequency scaling of kind "yarn" takes as trained on


# ---------------------------------------------------------------- cases


def _rot(dim, rot=None, interleaved=False, theta=10000.0, scaling="none", factor=1.0):
    """How heads are rotated: the first `rot` elements, pairs (i, i + rot / 2) or (2 i, 2 i + 1)."""
    return {"dim": dim, "rot": dim if rot is None else rot, "interleaved": interleaved, "theta": theta,
            "scaling": scaling, "factor": factor}


def _rotary(name, batch, tokens, heads, kv_heads, dtype, start, backward, **rot):
    c = {"kind": "rotary", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dtype": dtype,
         "start": start, "backward": backward, **_rot(**rot)}
    return {"name": name, **c} if name else c


def _append(name, seqs, chunk, singles, context, heads, kv_heads, page, dtype, **rot):
    """`seqs` sequences; round(singles * seqs) of them take one new token, the others up to `chunk`."""
    c = {"kind": "append", "seqs": seqs, "chunk": chunk, "singles": singles, "context": context, "heads": heads,
         "kv_heads": kv_heads, "page": page, "dtype": dtype, **_rot(**rot)}
    return {"name": name, **c} if name else c


def _attn(name, seqs, chunk, singles, context, heads, kv_heads, dim, page, dtype, window=-1, ratio=1.0):
    """window -1: every earlier key; ratio below 1: the share of new tokens whose gate selects them."""
    c = {"kind": "attn", "seqs": seqs, "chunk": chunk, "singles": singles, "context": context, "heads": heads,
         "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "window": window, "ratio": ratio}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a decode step of a few users far into their contexts: launches count
        _rotary("rotary_decode", 8, 1, 16, 16, "bf16", 900000, False, dim=128),
        # a training batch of the 1.5B model's heads with grouped keys, and its backward pass
        _rotary("rotary_train", 4, 8192, 16, 4, "bf16", 0, True, dim=128),
        # full precision, a quarter of an odd-sized head rotated, neighbouring pairs, a context scaled to eight times
        _rotary("rotary_fp32_part", 2, 5003, 8, 8, "fp32", 40000, True, dim=80, rot=20, interleaved=True, theta=500000.0,
                scaling="yarn", factor=8.0),
        # one token of each of 32 users into their pages
        _append("append_decode", 32, 1, 1.0, 2000, 16, 16, 16, "bf16", dim=128),
        # ragged prompt chunks beside single tokens, grouped heads, half of the head rotated by neighbouring pairs
        _append("append_chunks", 12, 4001, 0.34, 4000, 16, 4, 64, "fp16", dim=128, rot=64, interleaved=True,
                scaling="ntk", factor=4.0),
        # the smallest call: one token of one user
        _attn("attn_one_token", 1, 1, 1.0, 700, 16, 4, 128, 16, "bf16"),
        # a decode step of the global branch: long contexts, about half of the rows selected by their gates
        _attn("attn_decode_gated", 32, 1, 1.0, 16384, 16, 16, 128, 64, "bf16", ratio=0.5),
        # few users with very long contexts, eight query heads to a key head
        _attn("attn_decode_grouped", 3, 1, 1.0, 100003, 32, 4, 128, 16, "fp16"),
        # a step of a server: single tokens beside chunks of prompts, odd lengths
        _attn("attn_mixed", 16, 509, 0.75, 8191, 16, 4, 64, 32, "bf16"),
        # the local branch of prompt chunks
        _attn("attn_local", 4, 2048, 0.0, 6000, 16, 16, 128, 64, "bf16", window=128),
        # the global branch of a prompt's next chunk, a quarter of its tokens selected
        _attn("attn_selected", 1, 8192, 0.0, 24576, 16, 16, 128, 128, "bf16", ratio=0.25),
        # every token of the second half of a long prompt, grouped heads
        _attn("attn_prefill", 1, 16384, 0.0, 16384, 16, 4, 128, 64, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_rot(rng, dims):
    dim = rng.choice(dims)
    scaling = rng.choice(("none", "none", "linear", "ntk", "yarn"))
    return {"dim": dim, "rot": rng.choice((dim, dim, dim // 2, dim // 4)), "interleaved": rng.random() < 0.4,
            "theta": rng.choice((10000.0, 500000.0)), "scaling": scaling,
            "factor": 1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0))}


def draw(rng):
    kind = rng.choice(("rotary", "append", "attn", "attn"))
    heads = rng.choice((4, 8, 16, 32))
    kv_heads = heads // rng.choice((1, 1, 2, 4))
    if kind == "rotary":
        return _rotary(None, rng.randint(1, 4), _log(rng, 1, 4096), heads, kv_heads,
                       rng.choice(("bf16", "bf16", "fp16", "fp32")), _log(rng, 1, 1000000), rng.random() < 0.6,
                       **_draw_rot(rng, (64, 80, 128, 256)))
    seqs = _log(rng, 1, 48)
    singles = rng.choice((0.0, 0.5, 1.0, 1.0)) if kind == "attn" else rng.choice((0.0, 0.5, 1.0))
    page, dtype = rng.choice((16, 32, 64, 128)), rng.choice(("bf16", "bf16", "fp16"))
    if kind == "append":
        return _append(None, seqs, _log(rng, 1, 16384 // seqs), singles, _log(rng, 1, 49152 // seqs), heads, kv_heads,
                       page, dtype, **_draw_rot(rng, (64, 128)))
    chunk, context = _log(rng, 1, 16384 // seqs), _log(rng, 1, 262144 // seqs)
    c = _attn(None, seqs, chunk, singles, context, heads, kv_heads, rng.choice((64, 128, 128)), page, dtype,
              window=rng.choice((-1, -1, -1, 128, 1000)), ratio=rng.choice((1.0, 1.0, 0.25, 0.6)))
    top = work(listed()[-1])["flops"]
    while work(c)["flops"] > top:
        c["context"] = max(1, c["context"] // 2)
        c["chunk"] = max(1, c["chunk"] * 3 // 4)
    return c


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(shape, gen, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _lengths(case):
    """New tokens and cached ones before them of each sequence, fixed by the case: the first single and the first
    chunk have the longest context, the largest chunk is `chunk`."""
    n = case["seqs"]
    rs = np.random.RandomState(31 * n + case["chunk"] % 1009 + 7 * (case["context"] % 1013))
    one = int(round(case["singles"] * n))
    new = np.ones(n, dtype=np.int64)
    ctx = (rs.uniform(0.25, 1.0, n) * case["context"]).astype(np.int64)
    ctx[0] = case["context"]
    if one < n:
        new[one:] = np.maximum(1, (rs.uniform(0.3, 1.0, n - one) * case["chunk"]).astype(np.int64))
        new[one] = case["chunk"]
        ctx[one] = case["context"]
    return new, ctx


def _spans(n, ratio, rng):
    """A selection in spans of mean length 8, with gaps that give `ratio`."""
    run, gap = 8.0, 8.0 * (1.0 - ratio) / ratio
    count = int(2 * n / (run + gap)) + 16
    parts = np.empty(2 * count, dtype=np.int64)
    parts[0::2] = rng.geometric(1.0 / run, count)
    parts[1::2] = rng.geometric(1.0 / max(gap, 1.0), count)
    sel = np.repeat(np.tile([True, False], count), parts)
    return np.concatenate([sel, np.zeros(max(0, n - sel.size), dtype=bool)])[:n]


def _cache(case, gen, seed):
    """Pages in the order in which a server's free list hands them out after a while: any."""
    dt, page, h, d = DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["dim"]
    new, ctx = _lengths(case)
    lens = new + ctx
    need = -(-lens // page)
    total = int(need.sum()) + 3
    order = np.random.RandomState(int(seed) % (1 << 31)).permutation(total)
    table = np.zeros((len(lens), int(need.max())), dtype=np.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += int(k)
    cu = np.concatenate([[0], np.cumsum(new)])
    return {"new": new.tolist(), "lens": lens.tolist(), "n": int(cu[-1]), "max_q": int(new.max()),
            "max_len": int(lens.max()),
            "k_pages": _randn((total, h, page, d), gen, dt), "v_pages": _randn((total, h, page, d), gen, dt),
            "table": torch.from_numpy(table).to(DEV), "cu": torch.tensor(cu, dtype=torch.int32, device=DEV),
            "len": torch.tensor(lens, dtype=torch.int32, device=DEV)}


def _plan(case):
    from logo_amd.ops.rotary import rotary_plan

    scaling = None if case["scaling"] == "none" else case["scaling"]
    return rotary_plan(case["dim"], theta=case["theta"], rot_dim=case["rot"], interleaved=case["interleaved"],
                       scaling=scaling, factor=case["factor"], trained_len=TRAINED_LEN, device=DEV)


def prepare(case, seed):
    gen, dt, d = _gen(seed), DTYPES[case["dtype"]], case["dim"]
    if case["kind"] == "rotary":
        b, t = case["batch"], case["tokens"]
        first = torch.from_numpy(np.random.RandomState(int(seed) % (1 << 31)).randint(0, case["start"] + 1, (b, 1)))
        s = {"positions": (first + torch.arange(t)[None]).to(device=DEV, dtype=torch.int32),
             "q": _randn((b, t, case["heads"], d), gen, dt), "k": _randn((b, t, case["kv_heads"], d), gen, dt)}
        if case["backward"]:
            s["gq"], s["gk"] = _randn(s["q"].shape, gen, dt), _randn(s["k"].shape, gen, dt)
            s["q"].requires_grad_()
            s["k"].requires_grad_()
    elif case["kind"] == "append":
        s = _cache(case, gen, seed)
        h, hk = case["heads"], case["kv_heads"]
        rows = _randn((s["n"], (h + 2 * hk) * d), gen, dt)  # a stacked projection's rows [q | k | v]
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in rows.split((h * d, hk * d, hk * d), dim=1))
    else:
        s = _cache(case, gen, seed)
        s["q"] = _randn((s["n"], case["heads"], d), gen, dt)
        s["sel"] = None
        if case["ratio"] < 1.0:
            rng = np.random.RandomState((int(seed) + 1) % (1 << 31))
            sel = _spans(s["n"], case["ratio"], rng) if s["max_q"] > 1 else rng.rand(s["n"]) < case["ratio"]
            s["sel"] = torch.from_numpy(sel).to(DEV)
    if own and case["kind"] != "attn":
        s["plan"] = _plan(case)
    s["case"] = case
    return s


# ---------------------------------------------------------------- one pass


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "append": _own_append, "attn": _own_attn}[kind](state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attn": _plain_attn}[kind](state)


def _own_rotary(s):
    from logo_amd.ops.rotary import rotary

    if not s["case"]["backward"]:
        return tuple(rotary([s["q"], s["k"]], s["positions"], s["plan"]))
    q, k = rotary([s["q"], s["k"]], s["positions"], s["plan"])
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"])))


def _own_append(s):
    from logo_amd.ops.paged import paged_append

    q = paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["len"], q=s["q"],
                     plan=s["plan"])
    return q, s["k_pages"], s["v_pages"]


def _own_attn(s):
    from logo_amd.ops.paged import paged_attn

    w = s["case"]["window"]
    return paged_attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["len"], max_q=s["max_q"],
                      max_len=s["max_len"], window=w if w >= 0 else None, selection=s["sel"])


def _frequencies(case):
    """Radians per position of each pair, float64, and the factor on the rotated elements."""
    r, s, theta = case["rot"], case["factor"], case["theta"]
    i = np.arange(0, r, 2, dtype=np.float64) / r
    if case["scaling"] == "ntk" and r > 2:
        theta = theta * s ** (r / (r - 2))
    f = theta ** -i
    if case["scaling"] == "linear":
        return f / s, 1.0
    if case["scaling"] == "yarn":
        keep = np.clip((TRAINED_LEN * f / (2 * math.pi) - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return f * keep + f / s * (1.0 - keep), 0.1 * math.log(s) + 1.0
    return f, 1.0


def _cos_sin(case, positions):
    """cos and sin [..., 1, rot / 2] in 64 bits: far positions lose their angle in 32."""
    f, m = _frequencies(case)
    a = positions.double()[..., None, None] * torch.from_numpy(f).to(DEV)
    return torch.cos(a) * m, torch.sin(a) * m


def _rotate(case, x, cos, sin):
    """x [..., H, D] rotated in 32 bits, rounded once."""
    r = case["rot"]
    xf, cos, sin = x.float(), cos.float(), sin.float()
    y = xf.clone()
    if case["interleaved"]:
        a, b = xf[..., 0:r:2], xf[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = xf[..., :r // 2], xf[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return y.to(x.dtype)


@torch.no_grad()
def _plain_rotary(s):
    case = s["case"]
    cos, sin = _cos_sin(case, s["positions"])
    out = [_rotate(case, s[x], cos, sin) for x in ("q", "k")]
    if case["backward"]:
        out += [_rotate(case, s[g], cos, -sin) for g in ("gq", "gk")]
    return tuple(out)


def _new_positions(s):
    """Sequence and position of every new token, on the GPU."""
    new = s["cu"][1:] - s["cu"][:-1]
    seq = torch.repeat_interleave(torch.arange(len(s["new"]), device=DEV), new, output_size=s["n"])
    return seq, torch.arange(s["n"], device=DEV) - s["cu"][:-1][seq] + (s["len"] - new)[seq]


@torch.no_grad()
def _plain_append(s):
    case = s["case"]
    seq, pos = _new_positions(s)
    cos, sin = _cos_sin(case, pos)
    page, slot = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    s["k_pages"][page, :, slot] = _rotate(case, s["k"], cos, sin)
    s["v_pages"][page, :, slot] = s["v"]
    return _rotate(case, s["q"], cos, sin), s["k_pages"], s["v_pages"]


@torch.no_grad()
def _plain_attn(s):
    case = s["case"]
    h, d, page, w = case["kv_heads"], case["dim"], case["page"], case["window"]
    g = case["heads"] // h
    out = torch.zeros_like(s["q"])
    lo = 0
    for b, (n, length) in enumerate(zip(s["new"], s["lens"])):
        ids = s["table"][b, :-(-length // page)].long()
        k, v = (p[ids].transpose(0, 1).reshape(h, -1, d)[:, :length].float() for p in (s["k_pages"], s["v_pages"]))
        kt = k.transpose(1, 2).contiguous()
        step = max(1, (1 << 28) // (h * g * length))
        for r0 in range(0, n, step):
            rows = torch.arange(lo + r0, lo + min(n, r0 + step), device=DEV)
            pos = rows - lo + length - n
            first = max(0, length - n + r0 - w) if w >= 0 else 0  # no row of the step sees an earlier key
            last = length - n + min(n, r0 + step)
            q = s["q"][rows].float().reshape(-1, h, g, d).permute(1, 2, 0, 3).reshape(h, -1, d)
            p = torch.matmul(q, kt[:, :, first:last]).reshape(h, g, len(rows), -1) * d ** -0.5
            keys = torch.arange(first, last, device=DEV)
            hidden = keys[None] > pos[:, None]
            if w >= 0:
                hidden |= keys[None] < pos[:, None] - w
            p.masked_fill_(hidden, -math.inf)
            p.sub_(p.amax(-1, keepdim=True)).exp_()
            p.div_(p.sum(-1, keepdim=True))
            o = torch.matmul(p.reshape(h, -1, last - first), v[:, first:last])
            o = o.reshape(h * g, len(rows), d).transpose(0, 1).to(out.dtype)
            out[rows] = o if s["sel"] is None else o * s["sel"][rows][:, None, None]
        lo += n
    return out


# ---------------------------------------------------------------- what a pass cannot do without


def _seen_keys(length, n, w, share):
    """Visible (token, key) pairs and keys read of a sequence's n new tokens, at the mean share of selected tokens."""
    if w < 0:
        return share * (n * (length - n) + n * (n + 1) / 2), length
    pos = np.arange(length - n, length)
    return share * float(np.minimum(pos + 1, w + 1).sum()), min(length, n + w)


def work(case):
    size, d = 4 if case["dtype"] == "fp32" else 2, case["dim"]
    if case["kind"] == "rotary":
        n = case["batch"] * case["tokens"]
        passes = 2 if case["backward"] else 1
        rows = n * (case["heads"] + case["kv_heads"])
        return {"bytes": passes * (2 * rows * d * size + 4 * n), "flops": passes * 3 * rows * case["rot"]}
    new, ctx = _lengths(case)
    n = int(new.sum())
    if case["kind"] == "append":
        rows = n * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * (rows + n * case["kv_heads"]) * d * size + 8 * len(new), "flops": 3 * rows * case["rot"]}
    pairs = keys = 0.0
    for k, c in zip(new.tolist(), ctx.tolist()):
        p, r = _seen_keys(k + c, k, case["window"], case["ratio"])
        pairs += p
        keys += r * (case["ratio"] if k == 1 else 1.0)  # a single token that is not selected reads no key
    return {"bytes": (n * case["heads"] * (1 + case["ratio"]) + 2 * keys * case["kv_heads"]) * d * size,
            "flops": 4 * d * case["heads"] * pairs}


# ---------------------------------------------------------------- 64-bit results


def _turned(case, x, positions, sign=1.0):
    """x rotated in 64 bits, each pair as a complex number."""
    f, m = _frequencies(case)
    r = case["rot"]
    x = x.detach().double()
    part = x[..., :r]
    pair = part.unflatten(-1, (r // 2, 2)) if case["interleaved"] else part.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_complex(pair.contiguous())
    angle = sign * positions.double()[..., None, None] * torch.from_numpy(f).to(DEV)
    z = torch.view_as_real(z * torch.polar(torch.full_like(angle, m), angle))
    z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., r:]), dim=-1)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        out = [_turned(case, s[x], s["positions"]) for x in ("q", "k")]
        if case["backward"]:
            out += [_turned(case, s[g], s["positions"], -1.0) for g in ("gq", "gk")]
        return tuple(out)
    starts = np.concatenate([[0], np.cumsum(s["new"])])
    if case["kind"] == "append":
        pos = torch.from_numpy(np.concatenate([np.arange(t - n, t) for n, t in zip(s["new"], s["lens"])])).to(DEV)
        table, page = s["table"].cpu().numpy(), case["page"]
        flat = np.concatenate([table[b][np.arange(t - n, t) // page].astype(np.int64) * page + np.arange(t - n, t) % page
                               for b, (n, t) in enumerate(zip(s["new"], s["lens"]))])
        flat = torch.from_numpy(flat).to(DEV)
        pages = []
        for pool, rows in ((s["k_pages"], _turned(case, s["k"], pos)), (s["v_pages"], s["v"].double())):
            slots = pool.double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
            slots[flat] = rows
            pages.append(slots.unflatten(0, (-1, page)).transpose(1, 2))
        return _turned(case, s["q"], pos), pages[0], pages[1]
    if work(case)["flops"] > 2e13:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group = case["heads"] // case["kv_heads"]
    for b, (n, t) in enumerate(zip(s["new"], s["lens"])):
        rows = torch.arange(starts[b], starts[b + 1], device=DEV)
        if s["sel"] is not None:
            rows = rows[s["sel"][rows]]
        if rows.numel() == 0:
            continue
        at = torch.arange(t, device=DEV)
        ids, slot = s["table"][b].long()[at // case["page"]], at % case["page"]
        for h in range(case["kv_heads"]):
            k, v = s["k_pages"][ids, h, slot].double(), s["v_pages"][ids, h, slot].double()
            for part in rows.split(max(1, (1 << 27) // (group * t))):
                p = (part - int(starts[b]) + t - n)[:, None, None]
                x = torch.einsum("nhd,kd->nhk", s["q"][part, h * group:(h + 1) * group].double(), k) / math.sqrt(case["dim"])
                seen = (at <= p) if case["window"] < 0 else (at <= p) & (at >= p - case["window"])
                x = torch.where(seen, x, torch.full_like(x, -math.inf))
                x = torch.softmax(x, dim=-1)
                out[part, h * group:(h + 1) * group] = torch.einsum("nhk,kd->nhd", x, v)
    return out
