"""The 64-bit statements of oracle/cache8.py against independent ones, on the CPU."""
import torch

from oracle import cache8


def test_e4m3_rounding_is_the_conversion_of_exact_numbers():
    """Every fp32 number between neighbours, at their middle and beside it; torch converts fp32 correctly."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), torch.tensor([0.0, 447.0, 448.0])])
    x = torch.cat([x, -x])
    want = x.float().to(torch.float8_e4m3fn).double()
    assert torch.equal(cache8.to_e4m3(x), want)
    assert torch.equal(cache8.to_e4m3(torch.tensor([1e9, -float("inf")], dtype=torch.float64)).abs(),
                       torch.full((2,), 448.0, dtype=torch.float64))


def test_scale_is_the_least_power_of_two():
    for most in (448.0, 448.0000001, 447.0, 1.75, 1.7500001, 3e-39, 0.0, 3e38):
        s = cache8.scale_for(torch.tensor([most, float("inf"), float("nan")], dtype=torch.float64))
        assert most <= 448 * s and (s == 2.0 ** -126 or most > 448 * s / 2)


def test_backward_against_autograd_in_64_bits():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 5, 32, generator=gen, dtype=torch.float64)
    w = torch.randn(32, generator=gen, dtype=torch.float64)
    g = torch.randn(2, 3, 5, 32, generator=gen, dtype=torch.float64)
    ang = torch.randn(40, 8, generator=gen, dtype=torch.float64)
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(0, 40, (2, 5), generator=gen)
    for inter in (False, True):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        r = torch.rsqrt(a.square().mean(-1, keepdim=True) + 1e-6)
        y = cache8._rotate(a * r * b, cos[pos][:, None], sin[pos][:, None], inter)
        assert torch.allclose(y, cache8.norm_rotary(x, w, cos, sin, pos, inter), rtol=1e-12, atol=1e-12)
        da, db = torch.autograd.grad(y, (a, b), g)
        dx, dw, _, _ = cache8.norm_rotary_backward(x, w, g, cos, sin, pos, inter)
        assert torch.allclose(dx, da, rtol=1e-10, atol=1e-12) and torch.allclose(dw, db, rtol=1e-10, atol=1e-12)


def test_shipped_references_say_the_same():
    """flagattention_b200.testing in fp32 against the 64-bit statements: a rounding of the output apart."""
    import flagattention_b200 as fa
    gen = torch.Generator().manual_seed(3)
    q, k = torch.randn(2, 4, 9, 32, generator=gen).half(), torch.randn(2, 2, 9, 32, generator=gen).half()
    wq, wk = torch.randn(32, generator=gen), torch.randn(32, generator=gen)
    cos, sin = fa.rotary_tables(20, 16)
    pos = torch.randint(-2, 30, (2, 9), generator=gen)
    for inter in (False, True):
        y = fa.testing.qk_norm_rotary(q, k, wq, wk, cos, sin, pos, inter)
        for a, x, w in zip(y, (q, k), (wq, wk)):
            want = cache8.norm_rotary(x, w, cos, sin, pos, inter)
            # (half a step of fp16, and some twenty fp32 roundings of terms below 16)
            assert ((a.double() - want).abs() <= 2.0 ** -11 * want.abs() + 32 * 16 * 2.0 ** -24).all()
    codes = [torch.randn(7, 2, 16, 32, generator=gen).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.rand(7, 2, generator=gen) for _ in range(2)]
    bt = torch.randperm(7, generator=gen)[:6].view(2, 3)
    lens, qq = torch.tensor([40, 0]), torch.randn(2, 4, 32, generator=gen).half()
    got = fa.testing.paged_attention_8bit(qq, *codes, *scales, lens, bt, 0.2)
    want, size, _ = cache8.paged_attention_8bit(qq, *codes, *scales, lens, bt, 0.2)
    assert ((got.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -16 * size).all() and (got[1] == 0).all()
