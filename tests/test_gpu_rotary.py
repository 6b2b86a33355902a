"""GPU parity of the rotary embedding by positions against 64-bit arithmetic."""

import pytest
import torch

from logo_amd.ops.rotary import rotary, rotary_, rotary_plan
from tests import paged_ref as ref
from tests.helpers import gen

pytestmark = pytest.mark.gpu

PLANS = [
    dict(),
    dict(rot_dim=64),
    dict(rot_dim=2, interleaved=True),
    dict(interleaved=True, scaling="linear", factor=4.0),
    dict(scaling="ntk", factor=8.0, theta=500000.0),
    dict(rot_dim=32, interleaved=True, scaling="yarn", factor=4.0, trained_len=4096),
    dict(rot_dim=0),
]


def _freqs(D, kw):
    kw = {k: v for k, v in kw.items() if k not in ("rot_dim", "interleaved")}
    return kw


def _ref(x, pos, D, kw, inverse=False):
    rot = kw.get("rot_dim", D)
    f, amp = ref.frequencies(rot, **_freqs(D, kw))
    return ref.rotate(x, pos, rot, kw.get("interleaved", False), f, amp, inverse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kw", PLANS, ids=lambda k: "-".join(str(v) for v in k.values()) or "plain")
def test_rotary_and_gradients(gpu, dtype, kw):
    """Two tensors of different heads over [B, T], positions from negative to past 10^9."""
    D, g = 128, gen(1)
    x = [torch.randn(2, 37, h, D, generator=g).to(dtype) for h in (6, 1)]
    gy = [torch.randn(t.shape, generator=g).to(dtype) for t in x]
    pos = torch.randint(-70000, 1 << 30, (2, 37), generator=g, dtype=torch.int64)
    plan = rotary_plan(D, device=gpu, **kw)
    xs = [t.to(gpu).requires_grad_() for t in x]
    ys = rotary(xs, pos.to(gpu), plan)
    gx = torch.autograd.grad(ys, xs, [t.to(gpu) for t in gy])
    for t, y, gyt, gxt in zip(x, ys, gy, gx):
        r, mag = _ref(t, pos, D, kw)
        assert y.is_contiguous() and y.dtype == dtype
        ref.check("y", y, r, ref.rotate_bound(r, mag, dtype))
        r, mag = _ref(gyt, pos, D, kw, inverse=True)
        ref.check("dx", gxt, r, ref.rotate_bound(r, mag, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot,inter", [(80, 80, False), (80, 20, True), (80, 20, False), (96, 48, True), (2, 2, False),
                                         (6, 4, True), (100, 50, False), (256, 256, True), (256, 2, False), (256, 2, True), (256, 128, False), (1, 0, False)])
def test_head_dims_and_parts(gpu, dtype, D, rot, inter):
    """Every vector width, odd halves and the scalar form; one token and three."""
    for T in (1, 3):
        g = gen(D + rot + T)
        x = torch.randn(T, 5, D, generator=g).to(dtype)
        pos = torch.randint(0, 300000, (T,), generator=g, dtype=torch.int32)
        y, = rotary([x.to(gpu)], pos.to(gpu), rotary_plan(D, rot_dim=rot, interleaved=inter, device=gpu))
        f, _ = ref.frequencies(rot)
        r, mag = ref.rotate(x, pos, rot, inter, f)
        ref.check("y", y, r, ref.rotate_bound(r, mag, dtype))


def test_gradient_against_differences(gpu):
    """The map is linear, so in fp32 a difference quotient over a step of one has no truncation error; its rounding:
    two results of at most 8 and a sum of 2 * 384 products."""
    D, g = 64, gen(3)
    plan = rotary_plan(D, rot_dim=32, interleaved=True, scaling="yarn", factor=4.0, trained_len=100, device=gpu)
    x = torch.randn(2, 3, 2, D, generator=g).to(gpu).requires_grad_()
    w, d = (torch.randn(2, 3, 2, D, generator=g).to(gpu) for _ in range(2))
    pos = torch.tensor([5, 1000, 7], device=gpu)
    loss = lambda t: float((rotary([t], pos, plan)[0].double() * w.double()).sum())  # noqa: E731
    y, = rotary([x], pos, plan)
    y.backward(w)
    dif = loss(x.detach() + d) - loss(x.detach())
    assert abs(dif - float((x.grad.double() * d.double()).sum())) <= 768 * 8 * 4 * 2.0 ** -24


def test_second_derivative_and_partial_gradients(gpu):
    """The backward is the same operator, so it has a gradient itself; an output without one asks for no launch."""
    D, g = 64, gen(4)
    plan = rotary_plan(D, device=gpu)
    a, b, w = (torch.randn(1, 4, 2, D, generator=g).to(gpu).requires_grad_() for _ in range(3))
    pos = torch.arange(4, device=gpu)
    ya, yb = rotary([a, b], pos, plan)
    ga, = torch.autograd.grad(ya, a, w, create_graph=True)
    gw, = torch.autograd.grad(ga, w, torch.ones_like(ga))
    r, = rotary([torch.ones_like(ga)], pos, plan)
    assert torch.equal(gw, r)
    assert torch.autograd.grad(yb.sum(), b)[0].shape == b.shape


@pytest.mark.parametrize("inplace", [False, True])
def test_strides(gpu, inplace):
    """Column slices of stacked rows, [B, H, T, D] views, unaligned starts: the rows, and in place nothing beside them."""
    D, B, T, H = 64, 2, 9, 3
    g = gen(5)
    pos = torch.randint(0, 9000, (B, T), generator=g)
    plan = rotary_plan(D, rot_dim=32, device=gpu)
    f, _ = ref.frequencies(32)
    views = [
        lambda t: t(B, T, 2 * H * D)[..., H * D:].unflatten(-1, (H, D)),
        lambda t: t(B, H, T, D).transpose(1, 2),
        lambda t: t(B, T, H, D + 1)[..., 1:],
        lambda t: t(T, B, H, D).transpose(0, 1),
        lambda t: t(B, T, H, 2 * D)[..., 4:D + 4],
    ]
    for dtype in (torch.bfloat16, torch.float32):
        for view in views:
            store = {}
            x = view(lambda *s: store.setdefault("t", torch.randn(*s, generator=g).to(dtype).to(gpu)))
            before = store["t"].clone()
            r, mag = ref.rotate(x.cpu(), pos, 32, False, f)
            if inplace:
                assert rotary_([x], pos.to(gpu), plan)[0] is x
                y = x.clone()
                x.copy_(r.to(dtype).to(gpu))
                mask = torch.zeros_like(before)
                view(lambda *s: mask).fill_(1)
                assert torch.equal(store["t"][mask == 0], before[mask == 0])
            else:
                y, = rotary([x], pos.to(gpu), plan)
                assert torch.equal(store["t"], before)
            ref.check("y", y, r, ref.rotate_bound(r, mag, dtype))


def test_broadcast_positions_and_expanded_gradients(gpu):
    D, g = 64, gen(6)
    plan = rotary_plan(D, device=gpu)
    f, _ = ref.frequencies(D)
    x = torch.randn(3, 2, 5, 2, D, generator=g)
    pos = torch.arange(5, dtype=torch.int32) + 12345
    xg = x.to(gpu).requires_grad_()
    y, = rotary([xg], pos.to(gpu), plan)
    r, mag = ref.rotate(x, pos, D, False, f)
    ref.check("y", y, r, ref.rotate_bound(r, mag, torch.float32))
    y.sum().backward()  # the gradient that arrives has strides of zero
    r, mag = ref.rotate(torch.ones_like(x), pos, D, False, f, inverse=True)
    ref.check("dx", xg.grad, r, ref.rotate_bound(r, mag, torch.float32))


def test_empty_and_many_heads(gpu):
    plan = rotary_plan(64, device=gpu)
    empty, = rotary([torch.empty(0, 2, 64, device=gpu)], torch.empty(0, dtype=torch.int64, device=gpu), plan)
    assert empty.shape == (0, 2, 64)
    none, one = rotary([torch.empty(3, 0, 64, device=gpu), torch.ones(3, 1, 64, device=gpu)],
                       torch.zeros(3, dtype=torch.int64, device=gpu), plan)
    assert none.shape == (3, 0, 64) and bool((one == 1).all())
    x = torch.randn(3, 700, 64, generator=gen(7))
    pos = torch.tensor([1, 2, 3])
    f, _ = ref.frequencies(64)
    y, = rotary([x.to(gpu)], pos.to(gpu), plan)
    r, mag = ref.rotate(x, pos, 64, False, f)
    ref.check("y", y, r, ref.rotate_bound(r, mag, torch.float32))


def test_captured_training_pass_and_streams(gpu):
    """Forward and backward captured into a graph, replayed with eager work between, and run on a side stream."""
    D, g = 128, gen(8)
    plan = rotary_plan(D, device=gpu)
    x = torch.randn(2, 50, 4, D, generator=g).bfloat16().to(gpu).requires_grad_()
    gy = torch.randn(2, 50, 4, D, generator=g).bfloat16().to(gpu)
    pos = torch.arange(50, device=gpu)

    def step():
        y, = rotary([x], pos, plan)
        return y, torch.autograd.grad(y, x, gy)[0]

    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [t.detach().clone() for t in step()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = [t.detach() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        with torch.no_grad():
            x.mul_(1.25)
            gy.neg_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b), k
    assert not torch.equal(eager[0], out[0])


def test_in_place_writes(gpu):
    """The same tensor twice is refused; a tensor saved for a backward pass and rotated since is an error there."""
    plan = rotary_plan(64, device=gpu)
    x = torch.randn(1, 5, 2, 64, device=gpu)
    pos = torch.arange(5, device=gpu)
    with pytest.raises(ValueError, match="share memory"):
        rotary_([x, x], pos, plan)
    w = torch.ones(1, device=gpu, requires_grad=True)
    y = (x * w).sum()
    rotary_([x], pos, plan)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
