"""GPU parity of the paged append and the paged attention against 64-bit
arithmetic, on pools whose unused slots and pages hold NaN."""

import math

import pytest
import torch

from logo_amd.ops.paged import paged_append, paged_attn
from logo_amd.ops.rotary import rotary_plan
from tests import paged_ref as ref
from tests.helpers import gen

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _dev(ts, gpu):
    """The tensors on the device with their strides."""
    out = []
    for t in ts:
        d = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=gpu)
        out.append(d.copy_(t))
    return out


def _run(gpu, new, lens, HQ, H, D, page, dtype, seed, tail=0, select=None, order="page", **kw):
    g = gen(seed)
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, H, D, page, dtype, g, order=order)
    N = sum(new) + tail
    q = torch.randn(N, HQ, D, generator=g).to(dtype)
    sel = None
    if select is not None:
        sel = torch.rand(N, generator=g) < select
    r, mag = ref.paged_attn(q, kp, vp, table, cu, ln, selection=sel, **kw)
    args = [t.to(gpu) for t in (kp, vp, table, cu, ln)]
    o = paged_attn(q.to(gpu), *args, selection=None if sel is None else sel.to(gpu), max_q=max(new + [0]),
                   max_len=max(lens + [0]), **kw)
    ref.check("o", o, r, ref.attn_bound(r, mag, dtype))
    # bounds left to their defaults may cut the keys otherwise, within the same bound
    o2 = paged_attn(q.to(gpu), *args, selection=None if sel is None else sel.to(gpu), **kw)
    ref.check("o, default bounds", o2, r, ref.attn_bound(r, mag, dtype))
    return o


# lengths around tiles, pages and pieces; no keys before the chunk; a sequence without new tokens; one without keys
RAGGED = ([1, 0, 5, 33, 1, 64, 2], [1, 40, 5, 100, 700, 64, 1029])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("HQ,H,D,page", [(4, 4, 128, 16), (6, 2, 64, 32), (8, 1, 128, 64), (5, 1, 64, 16), (2, 2, 64, 1024)])
@pytest.mark.parametrize("kw", [dict(), dict(window=0), dict(window=37, select=0.5), dict(select=0.3, tail=7, scale=0.2)],
                         ids=lambda k: "-".join(k) or "plain")
def test_ragged(gpu, dtype, HQ, H, D, page, kw):
    _run(gpu, *RAGGED, HQ, H, D, page, dtype, seed=HQ + D, **kw)


@pytest.mark.parametrize("HQ,H,D", [(4, 4, 128), (8, 2, 64), (64, 1, 128), (40, 2, 128)])
@pytest.mark.parametrize("lens", [[1], [300, 31, 1000, 2], [5000, 4097]])
def test_single_tokens(gpu, HQ, H, D, lens):
    """A decode step: the keys of long rows are cut into pieces and joined."""
    _run(gpu, [1] * len(lens), lens, HQ, H, D, 16, BF16, seed=sum(lens))
    _run(gpu, [1] * len(lens), lens, HQ, H, D, 64, F16, seed=sum(lens) + 1, select=0.5, window=200)


@pytest.mark.parametrize("new,lens", [([130], [130]), ([257], [1300]), ([200, 1, 129], [900, 2000, 129]), ([513], [700])])
@pytest.mark.parametrize("kw", [dict(), dict(window=128), dict(select=0.25), dict(select=0.25, window=100)],
                         ids=lambda k: "-".join(k) or "plain")
@pytest.mark.parametrize("HQ,H,D", [(2, 2, 128), (4, 1, 64)])
def test_chunks(gpu, new, lens, kw, HQ, H, D):
    _run(gpu, new, lens, HQ, H, D, 16, BF16, seed=sum(new), **kw)


@pytest.mark.parametrize("order", ["page", "slot", "pair"])
def test_pool_and_query_strides(gpu, order):
    new, lens = RAGGED
    g = gen(11)
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 2, 64, 16, BF16, g, order=order)
    N = sum(new)
    rows = torch.randn(N, 3 * 4 * 64 + 8, generator=g).bfloat16()
    q = rows[:, 4 * 64:8 * 64].unflatten(1, (4, 64))
    r, mag = ref.paged_attn(q, kp, vp, table, cu, ln)
    rg = rows.to(gpu)
    qg = rg[:, 4 * 64:8 * 64].unflatten(1, (4, 64))
    wide = torch.full((table.shape[0], 2 * table.shape[1]), 7, dtype=torch.int32, device=gpu)
    wide[:, ::2] = table.to(gpu)
    for tb in (table.to(gpu), wide[:, ::2]):
        if order == "pair":
            both = torch.stack([kp, vp], dim=1).to(gpu)
            pools = [both[:, 0], both[:, 1]]
        else:
            pools = _dev([kp, vp], gpu)
        o = paged_attn(qg, *pools, tb, cu.to(gpu), ln.to(gpu), max_q=64, max_len=1029)
        ref.check("o", o, r, ref.attn_bound(r, mag, BF16))
    # heads before tokens, and rows at odd addresses
    qt = q.transpose(0, 1).contiguous().to(gpu).transpose(0, 1)
    odd = torch.empty(N * 4 * 64 + 1, dtype=BF16, device=gpu)[1:].view(N, 4, 64).copy_(q)
    for x in (qt, odd):
        o = paged_attn(x, *[t.to(gpu) for t in (kp, vp, table, cu, ln)], max_q=64, max_len=1029)
        ref.check("o", o, r, ref.attn_bound(r, mag, BF16))


def test_rows_of_no_sequence_and_of_no_key(gpu):
    """Rows behind the last sequence: zero, or left alone in a caller's out; tokens at negative positions see nothing;
    an unselected call reads nothing."""
    g = gen(12)
    new, lens = [4, 3, 40], [2, 0, 300]
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 2, 64, 16, BF16, g)
    N = sum(new) + 9
    q = torch.randn(N, 4, 64, generator=g).bfloat16()
    r, mag = ref.paged_attn(q, kp, vp, table, cu, ln)
    args = [t.to(gpu) for t in (kp, vp, table, cu, ln)]
    for bounds in (dict(max_q=40, max_len=300), dict(max_q=1, max_len=1), dict(max_q=40, max_len=4000), dict()):
        out = torch.full((N, 4, 64), 7.0, dtype=BF16, device=gpu)
        got = paged_attn(q.to(gpu), *args, out=out, **bounds)
        assert got is out and bool((out[sum(new):] == 7).all())
        ref.check("o", out[:sum(new)], r[:sum(new)], ref.attn_bound(r, mag, BF16)[:sum(new)])
        o = paged_attn(q.to(gpu), *args, **bounds)
        assert bool((o[sum(new):] == 0).all()) and bool((o[:2] == 0).all()) and bool((o[4:7] == 0).all())
        o = paged_attn(q.to(gpu), *args, selection=torch.zeros(N, dtype=torch.bool, device=gpu), **bounds)
        assert bool((o == 0).all())
    empty = torch.zeros(0, dtype=torch.int32, device=gpu)
    o = paged_attn(q.to(gpu), args[0], args[1], empty.view(0, 3), torch.zeros(1, dtype=torch.int32, device=gpu), empty)
    assert bool((o == 0).all())


def test_entries_that_name_no_page(gpu):
    """Keys of pages that the table does not name (freed behind a window, or out of range) are not seen."""
    g = gen(13)
    new, lens = [1, 20, 150], [500, 400, 600]
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 2, 128, 16, BF16, g)
    table[0, :20] = -1
    table[1, 3] = kp.shape[0]
    table[1, 7] = -2147483648
    table[2, 30:36] = 2147483647
    table[2, 0] = -5
    q = torch.randn(sum(new), 4, 128, generator=g).bfloat16()
    args = [t.to(gpu) for t in (kp, vp, table, cu, ln)]
    for kw in (dict(), dict(window=100)):
        r, mag = ref.paged_attn(q, kp, vp, table, cu, ln, **kw)
        for bounds in (dict(max_q=150, max_len=600), dict()):
            o = paged_attn(q.to(gpu), *args, **kw, **bounds)
            ref.check("o", o, r, ref.attn_bound(r, mag, BF16))


def test_large_scores_and_infinities(gpu):
    """Scores of thousands stay finite; a key of infinities or NaN spoils only the rows that see it."""
    g = gen(14)
    new, lens = [70], [200]
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 1, 64, 16, BF16, g)
    q = torch.randn(70, 2, 64, generator=g).bfloat16() * 40
    r, mag = ref.paged_attn(q, kp * 8, vp, table, cu, ln)
    args = [t.to(gpu) for t in (table, cu, ln)]
    o = paged_attn(q.to(gpu), (kp * 8).to(gpu), vp.to(gpu), *args)
    # |q| |k| scale is 320 times the bound's: 0.064 of sum p |v|, where two scores lie within it of each other
    ref.check("o", o, r, ref.half_step(BF16) * (mag + r.abs()) + 0.064 * mag)
    # query rows of NaN, keys and values of NaN and infinity at the chunk's last token
    r, mag = ref.paged_attn(q / 40, kp, vp, table, cu, ln)
    last = table[0, 199 // 16].item()
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2, q2 = kp.clone(), vp.clone(), q / 40
        k2[last, 0, 199 % 16] = bad
        v2[last, 0, 199 % 16] = bad
        q2[3] = math.nan
        for bounds in (dict(max_q=70, max_len=200), dict(max_len=100000)):
            o = paged_attn(q2.to(gpu), k2.to(gpu), v2.to(gpu), *args, **bounds).cpu()
            keep = [i for i in range(69) if i != 3]
            ref.check("o", o[keep], r[keep], ref.attn_bound(r, mag, BF16)[keep])
            assert bool(o[3].isnan().all())
            assert not bool(o[69].isfinite().any())


def test_streams_and_replays(gpu):
    """A decode step captured into two graphs that replay in turn, lengths growing on the device between replays."""
    g = gen(15)
    new, lens = [1, 1, 1], [900, 30, 1500]
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 2, 128, 16, BF16, g)
    q = torch.randn(3, 8, 128, generator=g).bfloat16().to(gpu)
    args = [t.to(gpu) for t in (kp, vp, table, cu, ln)]
    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        paged_attn(q, *args, max_q=1, max_len=1600)
        for w in (None, 64):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(paged_attn(q, *args, max_q=1, max_len=1600, window=w))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(4):
        for graph, out, w in zip(graphs, outs, (None, 64)):
            graph.replay()
            eager = paged_attn(q, *args, max_q=1, max_len=1600, window=w)
            torch.cuda.synchronize()
            assert torch.equal(out, eager) and bool(out.isfinite().all())
            r, mag = ref.paged_attn(q.cpu(), kp, vp, table, cu, ln - step, window=w)
            ref.check("o", out, r, ref.attn_bound(r, mag, BF16))
        args[4].sub_(1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("order", ["page", "slot", "pair"])
@pytest.mark.parametrize("kw", [None, dict(), dict(rot_dim=32, interleaved=True, scaling="ntk", factor=4.0)],
                         ids=["none", "plain", "part"])
def test_append(gpu, dtype, order, kw):
    """Every new key and value in its slot, every other slot as it was, q rotated; stacked [q | k | v] rows."""
    D, H, HQ = 64, 2, 4
    g = gen(16)
    new, lens = [1, 0, 5, 33, 1, 64, 2, 4], [1, 40, 5, 100, 700, 64, 1029, 2]
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, H, D, 16, dtype, g, order=order)
    table[6, 1028 // 16] = -1     # the last token's page is not held
    tail = 3
    N = sum(new) + tail
    rows = torch.randn(N, (HQ + 2 * H) * D, generator=g).to(dtype)
    q, k, v = (t.unflatten(1, (-1, D)) for t in rows.split((HQ * D, H * D, H * D), dim=1))
    pos = torch.cat([torch.arange(t - n, t) for n, t in zip(new, lens)] + [torch.zeros(tail, dtype=torch.int64)])
    rot = kw.get("rot_dim", D) if kw is not None else 0
    f, amp = ref.frequencies(rot, **{a: b for a, b in (kw or {}).items() if a in ("scaling", "factor")})
    inter = bool(kw and kw.get("interleaved"))
    rk, mk = ref.rotate(k, pos, rot, inter, f, amp)
    rq, mq = ref.rotate(q, pos, rot, inter, f, amp)
    if order == "pair":
        both = torch.stack([kp, vp], dim=1).to(gpu)
        kg, vg = both[:, 0], both[:, 1]
    else:
        kg, vg = _dev([kp, vp], gpu)
    plan = rotary_plan(D, device=gpu, **kw) if kw is not None else None
    rg = rows.to(gpu)
    qg, kn, vn = (t.unflatten(1, (-1, D)) for t in rg.split((HQ * D, H * D, H * D), dim=1))
    qo = paged_append(kn, vn, kg, vg, table.to(gpu), cu.to(gpu), ln.to(gpu), q=qg, plan=plan)
    gone = (pos < 0) | (torch.arange(N) >= sum(new))
    rq[gone], mq[gone] = 0, 0
    ref.check("q", qo, rq, ref.rotate_bound(rq, mq, dtype))
    kc, vc = kg.cpu(), vg.cpu()
    at = 0
    for s, n in enumerate(new):
        for i in range(n):
            p, t = lens[s] - n + i, at + i
            page = int(table[s, p // 16]) if p >= 0 else -1
            if page < 0:
                continue
            ref.check("k", kc[page, :, p % 16], rk[t], ref.rotate_bound(rk[t], mk[t], dtype))
            assert torch.equal(vc[page, :, p % 16], v[t])
            kc[page, :, p % 16], vc[page, :, p % 16] = kp[page, :, p % 16], vp[page, :, p % 16]
        at += n
    assert torch.equal(kc.view(torch.int16), kp.contiguous().view(torch.int16))
    assert torch.equal(vc.view(torch.int16), vp.contiguous().view(torch.int16))


def test_append_many_sequences_and_no_tokens(gpu):
    """More sequences than a wave has lanes, most of them without new tokens."""
    g = gen(17)
    new = [1 if i % 3 == 0 else 0 for i in range(200)]
    lens = [i % 50 + 1 for i in range(200)]
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 1, 128, 16, BF16, g)
    N = sum(new)
    k, v = (torch.randn(N, 1, 128, generator=g).bfloat16() for _ in range(2))
    args = [t.to(gpu) for t in (kp, vp, table, cu, ln)]
    assert paged_append(k.to(gpu), v.to(gpu), *args) is None
    t = 0
    for s, n in enumerate(new):
        if n:
            p = lens[s] - 1
            assert torch.equal(args[0][int(table[s, p // 16]), 0, p % 16].cpu(), k[t, 0])
            assert torch.equal(args[1][int(table[s, p // 16]), 0, p % 16].cpu(), v[t, 0])
            t += 1
    assert paged_append(k[:0].to(gpu), v[:0].to(gpu), *args) is None


def test_append_then_attend(gpu):
    """Prompts in chunks, then single tokens, as a server runs them: the same outputs as whole sequences in 64 bits."""
    g = gen(18)
    D, H, HQ, page = 64, 2, 4, 32
    total = [150, 70]
    plan = rotary_plan(D, device=gpu)
    f, _ = ref.frequencies(D)
    q, k, v = ([torch.randn(t, h, D, generator=g).bfloat16() for t in total] for h in (HQ, H, H))
    kp, vp = (torch.full((12, H, page, D), math.nan, dtype=BF16, device=gpu) for _ in range(2))
    table = torch.tensor([[3, 0, 11, 5, 7], [1, 9, 2, -1, -1]], dtype=torch.int32, device=gpu)
    done = [0, 0]
    outs = [[], []]
    for new in ([64, 0], [60, 33], [1, 36], [24, 1], [1, 0]):
        cu = torch.tensor([0, new[0], new[0] + new[1]], dtype=torch.int32, device=gpu)
        cut = lambda x: torch.cat([x[s][done[s]:done[s] + new[s]] for s in range(2)]).to(gpu)  # noqa: E731
        done_after = [d + n for d, n in zip(done, new)]
        lens = torch.tensor(done_after, dtype=torch.int32, device=gpu)
        qr = paged_append(cut(k), cut(v), kp, vp, table, cu, lens, q=cut(q), plan=plan)
        o = paged_attn(qr, kp, vp, table, cu, lens, max_q=max(new), max_len=max(done_after)).cpu()
        outs[0].append(o[:new[0]])
        outs[1].append(o[new[0]:])
        done = done_after
    assert done == total
    for s in range(2):
        t = total[s]
        pos = torch.arange(t)
        rot = lambda x: ref.rotate(x, pos, D, False, f)[0].to(BF16)  # noqa: E731  rounded where the kernel rounds
        pools = [torch.zeros(1, H, 256, D, dtype=BF16) for _ in range(2)]
        pools[0][0, :, :t], pools[1][0, :, :t] = rot(k[s]).transpose(0, 1), v[s].transpose(0, 1)
        r, mag = ref.paged_attn(rot(q[s]), *pools, torch.zeros(1, 1, dtype=torch.int32),
                                torch.tensor([0, t]), torch.tensor([t]))
        # a rotated value that fp32 puts on the other side of a rounding border is off by a whole step: at most a few,
        # each moving a score by 2^-7 of one of 64 products
        ref.check("o", torch.cat(outs[s]), r, ref.attn_bound(r, mag, BF16) + 2.0 ** -8 * mag)


@pytest.mark.parametrize("big", [False, True])
def test_many_sequences(gpu, big):
    """More sequences than a wave has lanes (and than the pieces are counted for), many of them empty."""
    g = gen(19)
    S = 150
    new = [0 if s % 4 == 3 else 1 + (s * 7) % (40 if big else 5) for s in range(S)]
    lens = [n + (s * 37) % 300 if s % 11 else n for s, n in enumerate(new)]
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 1, 64, 16, BF16, g)
    N = sum(new)
    q = torch.randn(N, 4, 64, generator=g).bfloat16()
    sel = torch.rand(N, generator=g) < 0.5
    args = [t.to(gpu) for t in (kp, vp, table, cu, ln)]
    for kw in (dict(), dict(window=30), dict(selection=sel)):
        r, mag = ref.paged_attn(q, kp, vp, table, cu, ln, **kw)
        kw = {k: v.to(gpu) if torch.is_tensor(v) else v for k, v in kw.items()}
        for bounds in (dict(max_q=max(new), max_len=max(lens)), dict(max_q=5, max_len=5000), dict()):
            o = paged_attn(q.to(gpu), *args, **kw, **bounds)
            ref.check("o", o, r, ref.attn_bound(r, mag, BF16))


@pytest.mark.parametrize("bounds", [dict(max_q=1, max_len=3000), dict(max_q=8, max_len=16), dict(max_q=100, max_len=1),
                                    dict(max_q=0, max_len=0), dict(max_q=100000, max_len=1 << 40)])
def test_wrong_bounds_cost_time_only(gpu, bounds):
    g = gen(20)
    new, lens = [40, 1, 9], [1500, 2999, 700]
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 2, 64, 32, F16, g)
    q = torch.randn(sum(new), 8, 64, generator=g).half()
    sel = torch.rand(sum(new), generator=g) < 0.6
    r, mag = ref.paged_attn(q, kp, vp, table, cu, ln, selection=sel)
    o = paged_attn(q.to(gpu), *[t.to(gpu) for t in (kp, vp, table, cu, ln)], selection=sel.to(gpu), **bounds)
    ref.check("o", o, r, ref.attn_bound(r, mag, F16))


@pytest.mark.parametrize("new,lens,cols", [([10, 3], [70, 50], 4), ([1, 1, 1], [40, 1100, 2000], 62), ([200, 5], [1400, 90], 75),
                                           ([150, 700], [2100, 2500], 131), ([2, 40], [33, 77], 0)])
@pytest.mark.parametrize("kw", [dict(), dict(window=20), dict(window=900)], ids=lambda k: str(k.get("window")))
def test_lens_beyond_the_table(gpu, new, lens, cols, kw):
    """Keys behind the block table have no page: tokens keep their positions and see what the table reaches."""
    g = gen(40)
    kp, vp, table, cu, ln = ref.paged_inputs(new, lens, 2, 64, 16, BF16, g)
    q = torch.randn(sum(new), 4, 64, generator=g).to(BF16)
    wide = table.clone()
    wide[:, cols:] = -1
    r, mag = ref.paged_attn(q, kp, vp, wide, cu, ln, **kw)
    pools = [kp.to(gpu), vp.to(gpu)]
    for bounds in ({}, dict(max_q=max(new), max_len=max(lens))):
        o = paged_attn(q.to(gpu), *pools, table[:, :cols].to(gpu), cu.to(gpu), ln.to(gpu), **bounds, **kw)
        ref.check("o", o, r, ref.attn_bound(r, mag, BF16))


@pytest.mark.parametrize("length", [1 << 30, (1 << 31) - 1])
@pytest.mark.parametrize("window", [None, 40, 1 << 30, 1 << 40])
@pytest.mark.parametrize("n,max_q", [(3, 3), (50, 50)])
def test_positions_up_to_32_bits(gpu, n, max_q, window, length):
    """Positions far behind the table: every key of the table is seen, or, with a window that ends behind it, none."""
    g = gen(43)
    kp, vp, table, cu, ln = ref.paged_inputs([n], [100], 2, 64, 16, BF16, g)
    table = table[:, :6]  # 96 keys
    q = torch.randn(n, 4, 64, generator=g).to(BF16)
    all_keys = window is None or window > length
    r, mag = ref.paged_attn(q, kp, vp, torch.nn.functional.pad(table, (0, 99), value=-1), cu, torch.tensor([1000]))
    part = window == 1 << 30 and length == 1 << 30  # the first keys: p - 2^30 < 0 for all tokens
    if not (all_keys or part):
        r, mag = torch.zeros_like(r), torch.zeros_like(mag)
    ln = torch.tensor([length], dtype=torch.int32, device=gpu)
    o = paged_attn(q.to(gpu), kp.to(gpu), vp.to(gpu), table.to(gpu), cu.to(gpu), ln, max_q=max_q, window=window)
    ref.check("o", o, r, ref.attn_bound(r, mag, BF16))


def test_pages_beyond_32_bits(gpu):
    """Pages 3 GB apart: element and byte offsets past 2^32."""
    D, H, page, stride = 64, 2, 16, 3 << 29
    pools = [torch.empty(2 * stride + H * page * D, dtype=BF16, device=gpu).as_strided(
        (3, H, page, D), (stride, page * D, D, 1)) for _ in range(2)]
    g = gen(21)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    cu, ln = torch.tensor([0, 40], dtype=torch.int32), torch.tensor([40], dtype=torch.int32)
    q, k, v = (torch.randn(40, h, D, generator=g).bfloat16() for h in (4, H, H))
    args = [*pools, table.to(gpu), cu.to(gpu), ln.to(gpu)]
    assert paged_append(k.to(gpu), v.to(gpu), *args) is None
    small = [torch.zeros(3, H, page, D, dtype=BF16) for _ in range(2)]
    for j in range(40):
        p = int(table[0, j // page])
        small[0][p, :, j % page], small[1][p, :, j % page] = k[j], v[j]
        assert torch.equal(pools[0][p, :, j % page].cpu(), k[j])
    r, mag = ref.paged_attn(q, *small, table, cu, ln)
    ref.check("chunk", paged_attn(q.to(gpu), *args, max_q=40, max_len=40), r, ref.attn_bound(r, mag, BF16))
    r, mag = r[39:], mag[39:]
    one = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    o = paged_attn(q[39:].to(gpu), *args[:3], one, args[4], max_q=1, max_len=40)
    ref.check("token", o, r, ref.attn_bound(r, mag, BF16))


def test_shared_pages_and_repeated_runs(gpu):
    """Two sequences with a common prefix in the same pages; the same call gives the same bits."""
    g = gen(22)
    kp, vp, table, cu, ln = ref.paged_inputs([3, 5], [800, 700], 2, 128, 64, BF16, g)
    table[1, :9] = table[0, :9]
    q = torch.randn(8, 6, 128, generator=g).bfloat16()
    r, mag = ref.paged_attn(q, kp, vp, table, cu, ln)
    args = [t.to(gpu) for t in (kp, vp, table, cu, ln)]
    for bounds in (dict(max_q=5, max_len=800), dict(max_q=50, max_len=800)):
        o = paged_attn(q.to(gpu), *args, **bounds)
        ref.check("o", o, r, ref.attn_bound(r, mag, BF16))
        for _ in range(5):
            assert torch.equal(o, paged_attn(q.to(gpu), *args, **bounds))


def test_append_captured_with_attention(gpu):
    """A decode step's append and attention in one graph, replayed as the lengths grow on the device."""
    D, H, HQ, page = 128, 2, 4, 16
    g = gen(23)
    plan = rotary_plan(D, rot_dim=64, interleaved=True, device=gpu)
    lens0 = [200, 5]
    kp, vp, table, _, ln = ref.paged_inputs([0, 0], lens0, H, D, page, BF16, g, spare=8)
    free = sorted(set(range(kp.shape[0])) - set(table.flatten().tolist()))
    table = torch.cat([table[:, :13], torch.full((2, 1), -1, dtype=torch.int32)], dim=1)
    table[0, 13], table[1, 1] = free[0], free[1]
    rows = torch.randn(2, (HQ + 2 * H) * D, generator=g).bfloat16().to(gpu)
    q, k, v = (t.unflatten(1, (-1, D)) for t in rows.split((HQ * D, H * D, H * D), dim=1))
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    twins = [[t.to(gpu) for t in (kp, vp, table, ln)] for _ in range(2)]

    def step(t):
        t[3].add_(1)
        qr = paged_append(k, v, t[0], t[1], t[2], cu, t[3], q=q, plan=plan)
        return paged_attn(qr, t[0], t[1], t[2], cu, t[3], max_q=1, max_len=220)

    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = [t.clone() for t in twins[0]]
        step(warm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(twins[0])
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(12):
        graph.replay()
        eager = step(twins[1])
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and bool(out.isfinite().all())
        rows.mul_(0.9)
    for a, b in zip(*twins):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())


def test_views_of_tables_and_pages(gpu):
    """One table for all sequences as an expanded view, a single page or head of any stride, results written over q."""
    g = gen(41)
    kp, vp, table, cu, ln = ref.paged_inputs([3, 2, 40], [90, 90, 90], 1, 64, 128, BF16, g)
    table[1:] = table[0]
    N = 45
    q = torch.randn(N, 4, 64, generator=g).to(BF16)
    r, mag = ref.paged_attn(q, kp, vp, table, cu, ln)
    page = int(table[0, 0])
    pools = []
    for p in (kp, vp):
        rows = torch.empty_strided((1, 1, 128, 64), (12345, 777, 64, 1), dtype=BF16, device=gpu)
        pools.append(rows.copy_(p[page:page + 1]))
    for big in (N, 8):  # both kernels
        tb = torch.zeros(1, 1, dtype=torch.int32, device=gpu).expand(3, 1)
        over = q.to(gpu)
        o = paged_attn(over, *pools, tb, cu.to(gpu), ln.to(gpu), max_q=big)
        ref.check("o", o, r, ref.attn_bound(r, mag, BF16))
        before = over._version
        assert paged_attn(over, *pools, tb, cu.to(gpu), ln.to(gpu), max_q=big, out=over) is over
        assert torch.equal(over, o) and over._version > before


def test_append_is_seen_by_autograd(gpu):
    """Pages saved for a backward pass and written since are an error there, as for any write in place."""
    g = gen(42)
    kp, vp, table, cu, ln = [t.to(gpu) for t in ref.paged_inputs([2], [20], 1, 64, 16, BF16, g)]
    w = torch.ones(1, device=gpu, dtype=BF16, requires_grad=True)
    y = (kp * w).sum()
    k = torch.randn(2, 1, 64, generator=g).to(BF16).to(gpu)
    paged_append(k, k, kp, vp, table, cu, ln)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        kp2, vp2 = kp.clone(), vp.clone()
        paged_append(k, k, kp2, vp2, table, cu, ln)


def test_operator_registrations(gpu):
    """torch.library's checks of the operators: schemas, fakes, autograd registration."""
    from logo_amd import _torch_ops

    ops = _torch_ops.ops()
    g = gen(24)
    kp, vp, table, cu, ln = (t.to(gpu) for t in ref.paged_inputs([3, 40], [30, 90], 1, 64, 16, BF16, g))
    kp, vp = kp.nan_to_num(), vp.nan_to_num()
    q = torch.randn(43, 2, 64, generator=g).bfloat16().to(gpu)
    k = torch.randn(43, 1, 64, generator=g).bfloat16().to(gpu)
    plan = rotary_plan(64, device=gpu)
    rot = (plan.turns, 64, 64, False, 1.0)
    check = torch.library.opcheck
    check(ops.paged_attn, (q, kp, vp, table, cu, ln, None, 40, 90, 0.125, -1))
    check(ops.paged_attn_out, (q, kp, vp, table, cu, ln, None, 40, 90, 0.125, -1, torch.empty_like(q)))
    check(ops.paged_append, (k, k.clone(), kp, vp, table, cu, ln, q, *rot))
    check(ops.paged_append, (k, k.clone(), kp, vp, table, cu, ln, None, None, 0, 0, False, 1.0))
    check(ops.rotary, ([q.float().requires_grad_()], torch.arange(43, device=gpu), *rot, False))
    check(ops.rotary_, ([q.clone()], torch.arange(43, device=gpu), *rot))
