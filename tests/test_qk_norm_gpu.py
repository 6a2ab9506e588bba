"""qk_norm_rotary against its definition in 64 bits, forward and backward.

Tolerances.  A result of fp32 arithmetic rounded once is off by half a step of its type, eps / 2 of its value (2^-24 more
where fp16 has no normal numbers), plus what fp32 loses: each operation 2^-24 of the sizes of its terms.  A rotated
element is two products of three factors, one of them r, whose sum of squares and reciprocal root come to some 40
roundings: 64 x 2^-24 of the terms' sizes bounds it.  dx has a second sum over the row: 128.  A sum of dw adds at most
8 rows a thread and position group, then groups: below 256 roundings at these sizes."""
import math

import pytest
import torch

import flagattention_b200 as fa
from oracle import cache8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def check(got, want, size, terms, what):
    half = torch.finfo(got.dtype).eps / 2
    least = 2.0 ** -25 if got.dtype == torch.float16 else 0.0      # half of fp16's smallest step
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    bound = half * want.abs() * (1 + half) + terms * U * size + least
    off = (got - want).abs() - bound
    assert off.max() <= 0, f"{what}: over its bound by {off.max():.3e} at {want.flatten()[off.argmax()]:.3e}"


def made(B, H, Hk, L, D, dtype, wdtype, R, layout, seed=0, rows=None):
    gen = torch.Generator().manual_seed(seed)

    def rnd(h):
        if layout == "bhld":
            return torch.randn(B, h, L, D, generator=gen).to(dtype).cuda()
        if layout == "blhd":
            return torch.randn(B, L, h, D, generator=gen).to(dtype).cuda().transpose(1, 2)
        # a slice of a wider projection
        return torch.randn(B, L, h, D + 16, generator=gen).to(dtype).cuda()[..., 8:D + 8].transpose(1, 2)

    q, k, gq, gk = rnd(H), rnd(Hk), rnd(H), rnd(Hk)
    wq, wk = (None, None) if wdtype is None else \
        ((1 + 0.3 * torch.randn(D, generator=gen)).to(wdtype).cuda() for _ in range(2))
    cos, sin = fa.rotary_tables(rows or L, R, device="cuda")
    return q, k, gq, gk, wq, wk, cos, sin


SHAPES = [  # B, H, Hk, L, D, R, layout
    (1, 1, 1, 1, 16, 16, "bhld"), (2, 3, 1, 5, 64, 64, "blhd"), (3, 4, 2, 37, 128, 128, "bhld"),
    (1, 8, 8, 130, 80, 32, "blhd"), (2, 5, 1, 33, 96, 96, "cut"), (1, 12, 4, 257, 128, 64, "cut"),
    (2, 2, 2, 19, 256, 256, "blhd"), (1, 3, 1, 9, 512, 512, "bhld"), (4, 17, 3, 66, 32, 16, "blhd"),
    (1, 2, 1, 70, 192, 96, "bhld"), (64, 32, 8, 1, 128, 128, "blhd"),
]


@pytest.mark.parametrize("B,H,Hk,L,D,R,layout", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.bfloat16, torch.bfloat16), (torch.float16, None)])
def test_forward_and_backward(B, H, Hk, L, D, R, layout, dtype, wdtype):
    inter = (L + H) % 2 == 1
    q, k, gq, gk, wq, wk, cos, sin = made(B, H, Hk, L, D, dtype, wdtype, R, layout)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk) if t is not None]
    yq, yk = fa.qk_norm_rotary(q, k, wq, wk, cos, sin, interleaved=inter)
    grads = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    for x, y, w, g, dx, n in ((q, yq, wq, gq, grads[0], 0), (k, yk, wk, gk, grads[1], 1)):
        assert y.dtype == dtype and y.shape == x.shape
        want = cache8.norm_rotary(x, w, cos, sin, None, inter)
        size = cache8.norm_rotary(x.abs(), None if w is None else w.abs(), cos.abs(), -sin.abs(), None, inter).abs() \
            .maximum(cache8.norm_rotary(x.abs(), None if w is None else w.abs(), cos.abs(), sin.abs(), None, inter).abs())
        check(y, want, size, 64, f"y{n}")
        want, dw, size, dw_size = cache8.norm_rotary_backward(x, w, g, cos, sin, None, inter)
        assert dx.dtype == dtype
        check(dx, want, size, 128, f"dx{n}")
        if w is not None:
            assert grads[2 + n].dtype == wdtype
            check(grads[2 + n], dw, dw_size, 256, f"dw{n}")


@pytest.mark.parametrize("shape", ["one row", "each its own"])
def test_positions_given_and_out_of_range(shape):
    B, H, Hk, L, D = 3, 4, 2, 21, 64
    q, k, gq, gk, wq, wk, cos, sin = made(B, H, Hk, L, D, torch.bfloat16, torch.float32, D, "bhld", rows=50)
    gen = torch.Generator().manual_seed(3)
    pos = torch.randint(-5, 60, (L,) if shape == "one row" else (B, L), generator=gen, dtype=torch.int32)
    q.requires_grad_()
    y, _ = fa.qk_norm_rotary(q, k, wq, wk, cos, sin, pos.cuda())
    dq, = torch.autograd.grad(y, q, gq)
    check(y, cache8.norm_rotary(q, wq, cos, sin, pos), cache8.norm_rotary(q.abs(), wq, cos.abs(), -sin.abs(), pos).abs()
          .maximum(cache8.norm_rotary(q.abs(), wq, cos.abs(), sin.abs(), pos).abs()), 64, "y")
    want, _, size, _ = cache8.norm_rotary_backward(q, wq, gq, cos, sin, pos)
    check(dq, want, size, 128, "dq")


def test_gradient_against_differences():
    """The analytic gradient of a 16-bit operator, against central differences of the 64-bit definition along a random
    direction: the directional derivative differs by the roundings of dx (half a step of each element)."""
    B, H, Hk, L, D = 2, 3, 1, 7, 64
    q, k, gq, gk, wq, wk, cos, sin = made(B, H, Hk, L, D, torch.float16, torch.float32, 32, "bhld")
    q.requires_grad_(), wq.requires_grad_()
    y, _ = fa.qk_norm_rotary(q, k, wq, wk, cos, sin)
    dq, dw = torch.autograd.grad(y, (q, wq), gq)
    gen = torch.Generator().manual_seed(5)
    for x, d, at in ((q, dq, 0), (wq, dw, 1)):
        v = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        h = 1e-5

        def f(t):
            xs = [q.detach().cpu().double(), wq.detach().cpu().double()]
            xs[at] = xs[at] + t * v
            return (cache8.norm_rotary(xs[0], xs[1], cos, sin) * gq.cpu().double()).sum()

        slope = (f(h) - f(-h)) / (2 * h)
        terms = d.detach().cpu().double() * v
        # half a step of each element; differences themselves: h^2 and 2^-52 / h, below 1e-8 of the terms
        assert abs(slope - terms.sum()) <= (torch.finfo(d.dtype).eps / 2 + 128 * U + 1e-8) * terms.abs().sum() + 1e-7


def test_layouts_agree_bit_for_bit_and_runs_repeat():
    B, H, Hk, L, D = 2, 6, 2, 300, 128
    q, k, gq, gk, wq, wk, cos, sin = made(B, H, Hk, L, D, torch.bfloat16, torch.float32, D, "bhld")
    runs = []
    for form in (lambda t: t, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: torch.cat((t, t), -1)[..., :D], lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
                 lambda t: torch.cat((t[..., :1], t), -1)[..., 1:], lambda t: t):
        leaves = [form(q).detach().requires_grad_(), form(k).detach().requires_grad_(),
                  wq.detach().requires_grad_(), wk.detach().requires_grad_()]
        y = fa.qk_norm_rotary(*leaves, cos, sin)
        runs.append([t.detach() for t in (*y, *torch.autograd.grad(y, leaves, (form(gq), form(gk))))])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_broadcast_operands_and_gradients():
    """k expanded over heads (stride 0) and a gradient that is one number expanded."""
    B, H, L, D = 2, 4, 40, 64
    q, k, _, _, wq, wk, cos, sin = made(B, H, 1, L, D, torch.float16, torch.float32, D, "bhld")
    k.requires_grad_(), wk.requires_grad_()
    wide = k.expand(B, H, L, D)
    y = fa.qk_norm_rotary(q, wide, wq, wk, cos, sin)
    dk, dwk = torch.autograd.grad(y[1].sum(), (k, wk))
    ref = fa.qk_norm_rotary(q, wide.detach().contiguous().requires_grad_(), wq, wk, cos, sin)
    assert torch.equal(y[1], ref[1])
    g = torch.ones(B, H, L, D, dtype=torch.float16)
    want, dw, size, dw_size = cache8.norm_rotary_backward(wide, wk, g, cos, sin)
    check(dwk, dw, dw_size, 256, "dwk")
    # torch adds the H heads' gradients in fp32 from values rounded to fp16, and rounds again
    half = 2.0 ** -11
    bound = half * want.abs().sum(1) + half * want.sum(1).abs() * (1 + H * half) + (128 + H) * U * size.sum(1) + H * 2.0 ** -24
    assert ((dk.cpu().double()[:, 0] - want.sum(1)).abs() <= bound).all()


def test_one_output_unused_and_frozen_weights():
    q, k, gq, gk, wq, wk, cos, sin = made(2, 4, 2, 33, 64, torch.bfloat16, torch.float32, 64, "bhld")
    q.requires_grad_(), k.requires_grad_(), wq.requires_grad_()
    y, _ = fa.qk_norm_rotary(q, k, wq, wk, cos, sin)
    dq, dk, dwq = torch.autograd.grad(y, (q, k, wq), gq, allow_unused=True)
    want, dw, size, dw_size = cache8.norm_rotary_backward(q, wq, gq, cos, sin)
    check(dq, want, size, 128, "dq")
    check(dwq, dw, dw_size, 256, "dwq")
    assert dk is None or (dk == 0).all()


def test_empty_calls():
    for B, L in ((0, 5), (2, 0)):
        q, k, gq, gk, wq, wk, _, _ = made(B, 4, 2, L, 64, torch.bfloat16, torch.float32, 64, "bhld")
        cos, sin = fa.rotary_tables(8, 64, device="cuda")
        for t in (q, k, wq, wk):
            t.requires_grad_()
        y = fa.qk_norm_rotary(q, k, wq, wk, cos, sin)
        assert y[0].shape == q.shape and y[1].shape == k.shape
        g = torch.autograd.grad(y, (q, k, wq, wk), (gq, gk))
        assert (g[2] == 0).all() and (g[3] == 0).all() and g[0].shape == q.shape


def test_extreme_rows():
    """A row of zeros stays 0 and has the gradient of eps; large values do not overflow on the way; a NaN stays in its row."""
    D = 64
    q = torch.randn(1, 1, 4, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    q[0, 0, 0] = 0
    q[0, 0, 1] *= 1e17
    q[0, 0, 2, 5] = float("nan")
    cos, sin = fa.rotary_tables(4, D, device="cuda")
    x = q.cuda().requires_grad_()
    y, _ = fa.qk_norm_rotary(x, x.detach(), None, None, cos, sin)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert (y[0, 0, 0] == 0).all() and torch.isnan(y[0, 0, 2]).all()
    keep = [0, 1, 3]
    want = cache8.norm_rotary(q, None, cos, sin)
    size = cache8.norm_rotary(q.abs(), None, cos.abs(), sin.abs()).abs().maximum(
        cache8.norm_rotary(q.abs(), None, cos.abs(), -sin.abs()).abs())
    check(y[:, :, keep], want[:, :, keep], size[:, :, keep], 64, "y")
    want, _, size, _ = cache8.norm_rotary_backward(q, None, torch.ones_like(q), cos, sin)
    check(dx[:, :, keep], want[:, :, keep], size[:, :, keep], 128, "dx")


def test_graph_capture_and_side_stream():
    """Run with its backward on a side stream, captured, and replayed on new values."""
    q, k, gq, gk, wq, wk, cos, sin = made(2, 4, 2, 100, 128, torch.bfloat16, torch.float32, 128, "bhld")
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    eager = fa.qk_norm_rotary(*leaves, cos, sin)
    want0 = [t.detach().clone() for t in (*eager, *torch.autograd.grad(eager, leaves, (gq, gk)))]
    del eager
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = fa.qk_norm_rotary(*leaves, cos, sin)
        side = [t.detach() for t in (*y, *torch.autograd.grad(y, leaves, (gq, gk)))]
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(side, want0))
    del y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fa.qk_norm_rotary(*leaves, cos, sin)
        out = [t for t in (*y, *torch.autograd.grad(y, leaves, (gq, gk)))]
    with torch.no_grad():
        q.copy_(q.flip(2))
        gk.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.detach().clone() for t in out]
    y2 = fa.qk_norm_rotary(*leaves, cos, sin)
    want = [t.detach() for t in (*y2, *torch.autograd.grad(y2, leaves, (gq, gk)))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_layer_trains():
    """qk_norm_rotary in front of flash_attention: gradients of a whole layer against the 32-bit PyTorch layer on the same
    16-bit operands, by the rule of the reference's tests (twice the error of the 16-bit PyTorch layer)."""
    from helpers import assert_within_2x
    B, H, Hk, L, D = 2, 8, 2, 200, 64
    q, k, gq, _, wq, wk, cos, sin = made(B, H, Hk, L, D, torch.bfloat16, torch.float32, D, "bhld")
    v = torch.randn(B, Hk, L, D, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    leaves = [t.requires_grad_() for t in (q, k, v, wq, wk)]
    o = fa.flash_attention(*fa.qk_norm_rotary(q, k, wq, wk, cos, sin), v, causal=True)
    got = (o, *torch.autograd.grad(o, leaves, gq))

    def layer(upcast):
        work = torch.float32 if upcast else torch.bfloat16

        def turn(x, w):
            x = x.to(work)
            x = (x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(work)) * w.to(work)
            a, b = x[..., :D // 2], x[..., D // 2:]
            c, s = cos.to(work), sin.to(work)
            return torch.cat((a * c - b * s, b * c + a * s), -1)

        return fa.testing.flash_attention(turn(q, wq), turn(k, wk), v.to(work), True, upcast=upcast).to(torch.bfloat16)

    sides = []
    for upcast in (True, False):
        o = layer(upcast)
        sides.append((o, *torch.autograd.grad(o, leaves, gq)))
    assert math.isfinite(got[0].float().sum().item())
    for name, h, r, t in zip(("o", "dq", "dk", "dv", "dwq", "dwk"), got, *sides):
        assert_within_2x(h, r, t, name)
