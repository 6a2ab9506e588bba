"""qk_norm_rotary and rotary_and_cache at sizes whose CTAs walk several heads, as prompts and training steps have them, with head
counts that leave the last CTA of a row fewer: the same definitions and tolerances as in the tests of small sizes.

Smaller calls leave a thread one or two heads (plan_norm() and launch_cache() fill the GPU first)."""
import pytest
import torch

import flagattention_b200 as fa
from test_rotary_cache_gpu import Batch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def turned(x, cos, sin, interleaved):
    """x (B, heads, L, D) in 64 bits on the GPU, cos and sin (L, R / 2)."""
    half = cos.shape[-1]
    y = x.clone()
    lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
    y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    return y


def near(got, want, size, terms, what):
    half = torch.finfo(got.dtype).eps / 2
    least = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    off = (got.detach().double() - want).abs() - half * want.abs() * (1 + half) - terms * U * size - least
    assert off.max() <= 0, f"{what}: over its bound by {off.max():.3e}"


@pytest.mark.parametrize("B,H,Hk,L,D,R,interleaved,layout,dtype", [
    (2, 5, 3, 12800, 64, 64, False, "bhld", torch.bfloat16),     # a thread has 5 heads forward; 2 backward, and one
    (3, 30, 3, 4300, 128, 64, True, "blhd", torch.float16),      # 16 and 14; 8 and 6
    (1, 17, 1, 1009, 256, 256, False, "blhd", torch.bfloat16),   # 2 and one; one
    (5, 11, 2, 2003, 80, 80, False, "bhld", torch.float16),      # 8 and 3; 4 and 3
])
def test_norm_and_rotation_of_many_heads(B, H, Hk, L, D, R, interleaved, layout, dtype):
    gen = torch.Generator(device="cuda").manual_seed(L)

    def rnd(h):
        shape = (B, h, L, D) if layout == "bhld" else (B, L, h, D)
        x = torch.randn(shape, generator=gen, device="cuda").to(dtype)
        return x if layout == "bhld" else x.transpose(1, 2)

    ws = [(1 + 0.3 * torch.randn(D, generator=gen, device="cuda")).requires_grad_() for _ in range(2)]
    xs, gs = [rnd(H).requires_grad_(), rnd(Hk).requires_grad_()], [rnd(H), rnd(Hk)]
    cos, sin = fa.rotary_tables(L, R, device="cuda")
    ys = fa.qk_norm_rotary(*xs, *ws, cos, sin, interleaved=interleaved)
    grads = torch.autograd.grad(ys, (*xs, *ws), gs)
    c, s = cos.double(), sin.double()
    for i in range(2):
        x, w, g = (t.detach().double() for t in (xs[i], ws[i], gs[i]))
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        n = x * r * w
        size = torch.maximum(*(turned(n.abs(), c.abs(), t, interleaved).abs() for t in (s.abs(), -s.abs())))
        near(ys[i], turned(n, c, s, interleaved), size, 64, f"y{i}")
        h = turned(g, c, -s, interleaved)
        h_size = torch.maximum(*(turned(g.abs(), c.abs(), t, interleaved).abs() for t in (s.abs(), -s.abs())))
        dx = r * (h * w - x * r * r * (h * w * x).mean(-1, keepdim=True))
        size = r * (h_size * w.abs() + x.abs() * r * r * (h_size * w.abs() * x.abs()).mean(-1, keepdim=True))
        near(grads[i], dx, size, 128, f"dx{i}")
        # a thread adds its part of a CTA's share one by one (135 at most: strips * heads / 592 CTAs), then come groups, warps
        # and rows of partial sums, 21; a term has some 45 roundings of its own: 256 bounds it
        near(grads[2 + i], (h * x * r).sum((0, 1, 2)), (h_size * x.abs() * r).sum((0, 1, 2)), 256, f"dw{i}")


@pytest.mark.parametrize("held", [True, False])
@pytest.mark.parametrize("T,Hq,Hk,D,BS,extra", [
    (2100, 20, 5, 128, 16, dict()),                                  # 8 bits: units of 4 heads and of one
    (10100, 20, 3, 128, 16, dict(norm=None, interleaved=True)),      # a thread has 8 heads of a row (4); units of 3
    (5100, 20, 5, 128, 64, dict(R=64)),                              # 4 (2); blocks of several passes
    (12000, 9, 6, 64, 16, dict(interleaved=True)),                   # 2 (1); units of 4 and of 2
])
def test_prompts_into_the_cache(T, Hq, Hk, D, BS, extra, held):
    gen = torch.Generator().manual_seed(T)
    new, past = [], []
    while sum(new) < T:
        new.append(min(int(torch.randint(1, 900, (1,), generator=gen)), T - sum(new)))
        past.append(int(torch.randint(0, 400, (1,), generator=gen)))
    b = Batch(past, new, Hq, Hk, D, BS, torch.bfloat16, held, seed=T, pad=37, **extra)
    if held:   # scales as a user's cache may have them, among powers of two
        for s in (b.ks, b.vs):
            odd = torch.rand(s.shape, generator=gen) < 0.3
            s[odd] = (0.1 + 3 * torch.rand(s.shape, generator=gen))[odd]
    d = b.device()
    b.check(b.call(d), d)
