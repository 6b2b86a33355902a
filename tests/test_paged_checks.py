"""Refusals of the paged cache's operators and of the rotary embedding, and the
rotary plan's frequencies (CPU: nothing is launched)."""

import ctypes
import math
import re

import pytest
import torch

from logo_amd import _lib
from logo_amd.ops.paged import paged_append, paged_attn
from logo_amd.ops.rotary import rotary, rotary_, rotary_plan
from tests import paged_ref as ref

BF16 = torch.bfloat16


@pytest.mark.parametrize("rot,kw", [
    (128, {}), (64, dict(theta=500000.0)), (128, dict(scaling="linear", factor=8.0)),
    (32, dict(scaling="ntk", factor=4.0)), (2, dict(scaling="ntk", factor=4.0)),
    (128, dict(scaling="yarn", factor=16.0, trained_len=4096)), (0, {}),
])
def test_plan_frequencies(rot, kw):
    """Turns per position in units of 2^-64, to the 53 bits of a float64."""
    plan = rotary_plan(128, rot_dim=rot, **kw)
    f, amp = ref.frequencies(rot, **kw)
    assert plan.turns.dtype == torch.int64 and plan.turns.shape == (rot // 2,) and plan.amplitude == pytest.approx(amp)
    for t, x in zip(plan.turns.tolist(), f.tolist()):
        assert (t % (1 << 64)) / 2.0 ** 64 == pytest.approx(x / (2 * math.pi), rel=1e-14)


def test_plan_turns_wrap():
    """A base below one has frequencies above a turn a position: they are taken modulo one."""
    plan = rotary_plan(4, theta=0.001)
    x = 0.001 ** -0.5 / (2 * math.pi)
    assert (plan.turns[1].item() % (1 << 64)) / 2.0 ** 64 == pytest.approx(x - math.floor(x), rel=1e-12)


@pytest.mark.parametrize("kw,msg", [
    (dict(head_dim=0), "head_dim"), (dict(head_dim=257), "head_dim"), (dict(head_dim=64, rot_dim=66), "rot_dim"),
    (dict(head_dim=64, rot_dim=31), "rot_dim"), (dict(head_dim=64, rot_dim=-2), "rot_dim"), (dict(head_dim=63), "rot_dim"),
    (dict(head_dim=64, theta=0.0), "theta"), (dict(head_dim=64, theta=math.inf), "theta"),
    (dict(head_dim=64, scaling="dynamic"), "scaling"), (dict(head_dim=64, scaling="linear", factor=0.0), "factor"),
    (dict(head_dim=64, scaling="yarn", factor=2.0), "trained_len"),
    (dict(head_dim=64, scaling="yarn", factor=0.5, trained_len=100), "factor"),
])
def test_plan_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        rotary_plan(**kw)


def test_rotary_refusals():
    plan = rotary_plan(64)
    x, pos = torch.zeros(2, 5, 3, 64), torch.arange(5)
    for xs, p, err, msg in (
            ([], pos, ValueError, "one to four"), ([x] * 5, pos, ValueError, "one to four"),
            ([x, x[:1]], pos, ValueError, "one type and shape"), ([x, x.half()], pos, ValueError, "one type"),
            ([x[..., :32]], pos, ValueError, "D = 64"), ([x[0, 0]], pos, ValueError, "T, H, D"),
            ([x.double()], pos, ValueError, "bf16, fp16 or fp32"), ([x], pos.float(), ValueError, "int32 or int64"),
            ([x], torch.arange(4), ValueError, "do not match"), ([x], torch.zeros(3, 2, 5).long(), ValueError, "do not match"),
            ([x], pos, RuntimeError, "no CPU fallback")):
        for fn in (rotary, rotary_):
            with pytest.raises(err, match=msg):
                fn(xs, p, plan)


def _args(S=2, P=6, H=2, page=16, D=64, M=3, N=5, HQ=4, dtype=BF16):
    return dict(q=torch.zeros(N, HQ, D, dtype=dtype), k_pages=torch.zeros(P, H, page, D, dtype=dtype),
                v_pages=torch.zeros(P, H, page, D, dtype=dtype), block_table=torch.zeros(S, M, dtype=torch.int32),
                cu_seqlens=torch.zeros(S + 1, dtype=torch.int32), lens=torch.zeros(S, dtype=torch.int32))


@pytest.mark.parametrize("change,msg", [
    (dict(v_pages=torch.zeros(6, 2, 16, 64)), "one shape and type"),
    (dict(v_pages=torch.zeros(6, 1, 16, 64, dtype=BF16)), "one shape and type"),
    (dict(block_table=torch.zeros(2, 3).long()), "int32"), (dict(lens=torch.zeros(2)), "int32"),
    (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), "do not match"),
    (dict(block_table=torch.zeros(3, 3, dtype=torch.int32)), "do not match"),
    (dict(block_table=torch.zeros(6, dtype=torch.int32)), "block_table must be"),
])
def test_cache_refusals(change, msg):
    a = {**_args(), **change}
    with pytest.raises(ValueError, match=msg):
        paged_attn(**a)
    q = a.pop("q")
    with pytest.raises(ValueError, match=msg):
        paged_append(q[:, :2], q[:, :2], **a)


@pytest.mark.parametrize("shape,msg", [(dict(D=32), "head dim"), (dict(D=256), "head dim"), (dict(page=8), "page_size"),
                                       (dict(page=48), "page_size"), (dict(dtype=torch.float32), "bf16 or fp16")])
def test_cache_shapes(shape, msg):
    with pytest.raises(ValueError, match=msg):
        paged_attn(**_args(**shape))


def test_cache_alignment():
    a = _args()
    a["k_pages"] = torch.zeros(6, 2, 16, 68, dtype=BF16)[..., :64]
    with pytest.raises(ValueError, match="16-byte aligned"):
        paged_attn(**a)
    a["k_pages"] = torch.zeros(6, 2, 64, 16, dtype=BF16).transpose(2, 3)
    with pytest.raises(ValueError, match="16-byte aligned"):
        paged_attn(**a)


@pytest.mark.parametrize("kw,msg", [
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"), (dict(window=-1), "window"),
    (dict(q=torch.zeros(5, 3, 64, dtype=BF16)), "multiple"), (dict(q=torch.zeros(5, 4, 64)), "q must be"),
    (dict(q=torch.zeros(5, 4, 128, dtype=BF16)), "q must be"), (dict(selection=torch.ones(5)), "selection"),
    (dict(selection=torch.ones(4, dtype=torch.bool)), "selection"), (dict(out=torch.zeros(5, 4, 64)), "out must be"),
    (dict(q=torch.zeros(5, 4, 64, dtype=BF16, requires_grad=True)), "no gradients"),
])
def test_attn_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        paged_attn(**{**_args(), **kw})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attn(**_args())


def test_shared_memory_refusals():
    """Memory that a call would write and read, or write twice."""
    a = _args()
    both = torch.zeros(5, 8, 64, dtype=BF16)
    with pytest.raises(ValueError, match="out overlaps"):
        paged_attn(**{**a, "q": both[:, 4:].transpose(0, 1).contiguous().transpose(0, 1), "out": a["k_pages"].view(-1)[:1280].view(5, 4, 64)})
    line = torch.zeros(2000, dtype=BF16)
    with pytest.raises(ValueError, match="out overlaps"):
        paged_attn(**{**a, "q": line[:1280].view(5, 4, 64), "out": line[64:1344].view(5, 4, 64)})
    for kw in (dict(v_pages=a["k_pages"]), dict(k_pages=a["k_pages"][:, :1].expand(6, 2, 16, 64)),
               dict(v_pages=a["k_pages"][:1].clone().expand(6, 2, 16, 64))):
        with pytest.raises(ValueError, match="share memory"):
            b = {**a, **kw}
            q = b.pop("q")
            paged_append(q[:, :2], q[:, :2], **b)
    for name in ("k_pages", "v_pages"):
        with pytest.raises(ValueError, match="no gradients"):
            paged_attn(**{**a, name: a[name].clone().requires_grad_()})


def test_append_refusals():
    a = _args()
    q = a.pop("q")
    k = q[:, :2]
    for kw, msg in ((dict(k=k[..., :32], v=k[..., :32]), "of the pages"), (dict(k=k.float(), v=k.float()), "of the pages"),
                    (dict(k=q, v=q), "of the pages"), (dict(k=k, v=k[:4]), "of the pages"), (dict(k=k, v=k, q=q[:4]), "q must"),
                    (dict(k=k, v=k, q=q.half()), "q must"), (dict(k=k, v=k, plan=rotary_plan(128)), "plan is for"),
                    (dict(k=k.clone().requires_grad_(), v=k), "no gradients")):
        with pytest.raises(ValueError, match=msg):
            paged_append(**kw, **a)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_append(k, k, **a)


def _cache(**kw):
    c = _lib.PagedCacheArg()
    vals = dict(k=256, v=256, k_page=2048, k_head=1024, k_slot=64, v_page=2048, v_head=1024, v_slot=64, pages=4, table=256,
                table_row=3, cu=256, lens=256, table_width=3, page_size=16, heads=2, nseq=2)
    for n, v in {**vals, **kw}.items():
        setattr(c, n, v)
    return c


@pytest.mark.parametrize("kw,msg", [
    (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(heads=0), "head count"),
    (dict(k_slot=60), "multiples of 8"), (dict(v_slot=56), "hold a row"), (dict(k=264), "16-byte"), (dict(k=None), "null"),
    (dict(table_row=2), "counts"), (dict(nseq=-1), "counts"), (dict(lens=None), "null"),
    (dict(table_width=1 << 27, table_row=1 << 27), "2\\^30"), (dict(k_slot=1 << 27), "2 GB"),
])
def test_c_entries_refuse_bad_caches(kw, msg):
    """Before any HIP call (pointers are placeholders)."""
    lib = _lib.lib()
    p = ctypes.c_void_p(256)
    c = _cache(**kw)
    assert lib.logo_paged_attn(c, p, 128, 64, p, None, 4, 5, 64, 1, 40, 0.1, -1, 1, p, 1 << 30, _lib.DTYPE_BF16, None) == 1
    assert re.search(msg, lib.logo_last_error().decode())
    assert lib.logo_paged_append(c, p, 128, 64, p, 128, 64, None, 0, 0, None, 0, 5, 64, None, 0, 0, 1.0, _lib.DTYPE_BF16,
                                 None) == 1
    assert re.search(msg, lib.logo_last_error().decode())


def test_c_entries_refuse_bad_arguments():
    lib = _lib.lib()
    p = ctypes.c_void_p(256)
    c = _cache()
    err = lambda: lib.logo_last_error().decode()  # noqa: E731
    attn = lambda q_tok=128, hq=4, n=5, d=64, scale=0.1, w=-1, dt=0, ws=p, nb=1 << 30: lib.logo_paged_attn(  # noqa: E731
        c, p, q_tok, 64, p, None, hq, n, d, 1, 4000, scale, w, 1, ws, nb, dt, None)
    for kw, msg in ((dict(hq=3), "multiple"), (dict(d=96), "head dim"), (dict(scale=0.0), "scale"), (dict(w=-2), "window"),
                    (dict(dt=1), "16-bit"), (dict(q_tok=4), "aligned"), (dict(n=1 << 30), "rows"), (dict(ws=None), "workspace"),
                    (dict(nb=16), "workspace")):
        assert attn(**kw) == 1 and msg in err(), kw
    rows = (_lib.Rows * 1)()
    rot = lambda n=1, bits=32, d=64, r=64, t=p, amp=1.0, dt=0: lib.logo_rotary(  # noqa: E731
        rows, n, p, bits, 5, 5, d, t, r, 0, amp, 0, dt, None)
    for kw, msg in ((dict(n=0), "one to four"), (dict(n=5), "one to four"), (dict(bits=16), "int32 or int64"),
                    (dict(d=257), "head dim"), (dict(r=33), "even"), (dict(r=66), "even"), (dict(t=None), "turns"),
                    (dict(amp=math.inf), "amplitude"), (dict(dt=5), "dtype"), (dict(), "null pointer")):
        assert rot(**kw) == 1 and msg in err(), kw
    assert lib.logo_paged_append(c, p, 128, 64, p, 128, 64, p, 256, 64, None, 4, 5, 64, None, 0, 0, 1.0, 0, None) == 1
    assert "output" in err()
