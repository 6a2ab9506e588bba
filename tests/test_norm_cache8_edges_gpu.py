"""Corners of qk_norm_rotary, rotary_and_cache and paged_attention_8bit, against their definitions in 64 bits: infinities beside
elements that only pass, batches cut short, scales that are no powers of two, the smallest scales, eps of 0."""
import pytest
import torch

import flagattention_b200 as fa
from oracle import cache8
from test_rotary_cache_gpu import E4M3, Batch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def same_where_not_finite(got, want):
    """NaN where the definition has NaN, infinities where it has those; returns where both are finite."""
    got, want = got.detach().cpu().double(), want.double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[got.isinf()], want[want.isinf()])
    return finite


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("held", [True, False])
@pytest.mark.parametrize("norm", [None, "fp32"])
@pytest.mark.parametrize("R", [32, 64])
def test_an_infinity_stays_among_the_elements_that_only_pass(R, norm, held, interleaved):
    """Partial rotation: an element behind the rotated ones has no partner, so an infinity or a NaN in it is its own affair.  With
    the norm its row's r is 0 (NaN) instead, for either form.

    Queries and 16-bit keys: half a step and the 64 roundings of test_rotary_cache_gpu.py, of the sizes of finite terms."""
    D = 128
    b = Batch([3, 0, 20], [18, 1, 5], 2, 2, D, 16, torch.bfloat16, held, R=R, norm=norm, seed=R, interleaved=interleaved)
    q, k, _ = b.parts(b.qkv)
    inf, nan = float("inf"), float("nan")
    for x in (q, k):
        x[1, 0, R + 3], x[2, 1, R], x[4, 0, D - 1], x[5, 1, R + 17] = inf, -inf, inf, nan
        x[18, 0, R + 8:R + 12] = inf
        x[20, 1, 5] = inf       # among the rotated ones: its pair
    d = b.device()
    out = b.call(d)
    want_q, kc, vc, ks, vs = b.expected()
    pairs = [(out, want_q)]
    if held:
        assert torch.equal(d["ks"].cpu().double(), ks) and torch.equal(d["vs"].cpu().double(), vs)
        got = d["kc"].cpu().view(E4M3).double()
        assert ((got == kc) | (got.isnan() & kc.isnan())).all()
    else:
        assert torch.equal(d["vc"].cpu().double(), vc)
        pairs.append((d["kc"], kc))
    b.qkv = torch.where(torch.isfinite(b.qkv), b.qkv, 0.0)
    sizes = b.expected(abs_=True)
    for (got, want), size in zip(pairs, sizes):
        ok = same_where_not_finite(got, want)
        if norm:   # (rows with an infinity or a NaN have r of 0 or NaN; the sizes are those of the row without it)
            assert ok.any()
        off = (got.cpu().double() - want).abs() - 2.0 ** -8 * want.abs() * (1 + 2.0 ** -8) - 64 * U * size
        assert off[ok].max() <= 0


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weights", [True, False])
def test_an_infinity_stays_in_its_element_of_norm_and_gradients(weights, interleaved):
    """The same of qk_norm_rotary: with an infinity in a row r is 0, and only the infinite element is NaN.  In the gradient of the
    result an infinity reaches its own column of the weight's gradient and no other."""
    B, H, L, D, R = 2, 3, 21, 96, 32
    gen = torch.Generator().manual_seed(1)
    x, g = (torch.randn(B, H, L, D, generator=gen).to(torch.bfloat16) for _ in range(2))
    w = 1 + 0.3 * torch.randn(D, generator=gen) if weights else None
    cos, sin = fa.rotary_tables(L, R)
    x[0, 1, 4, R + 5] = float("inf")
    x[1, 2, 20, D - 1] = -float("inf")
    x[1, 0, 3, R + 9] = float("nan")
    c = {n: None if t is None else t.cuda() for n, t in dict(x=x, w=w, cos=cos, sin=sin).items()}
    y, _ = fa.qk_norm_rotary(c["x"], c["x"], c["w"], c["w"], c["cos"], c["sin"], interleaved=interleaved)
    want = cache8.norm_rotary(x, w, cos, sin, None, interleaved)
    ok = same_where_not_finite(y, want)
    assert ok[0, 1, 4].sum() == D - 1 and ok[1, 2, 20].sum() == D - 1 and not ok[1, 0, 3].any()
    clean = torch.where(torch.isfinite(x), x, 0.0).abs()
    size = torch.maximum(*(cache8.norm_rotary(clean, None if w is None else w.abs(), cos.abs(), s, None, interleaved).abs()
                           for s in (sin.abs(), -sin.abs())))
    off = (y.cpu().double() - want).abs() - 2.0 ** -8 * want.abs() * (1 + 2.0 ** -8) - 64 * U * size
    assert off[ok].max() <= 0
    if w is None:
        return
    x = clean.float().to(torch.bfloat16) + 0.5
    g[1, 1, 7, R + 11] = float("inf")
    g[0, 0, 20, D - 8] = -float("inf")
    xs, ws = x.cuda().requires_grad_(), c["w"].requires_grad_()
    y, _ = fa.qk_norm_rotary(xs, xs.detach(), ws, c["w"].detach(), c["cos"], c["sin"], interleaved=interleaved)
    dw, = torch.autograd.grad(y, ws, g.cuda())
    _, want, _, size = cache8.norm_rotary_backward(x, w, torch.where(torch.isfinite(g), g, 0.0), cos, sin, None, interleaved)
    reached = torch.zeros(D, dtype=torch.bool)
    reached[[R + 11, D - 8]] = True
    assert torch.equal(dw.cpu().isfinite(), ~reached)
    assert ((dw.cpu().double() - want).abs() - 2.0 ** -24 * want.abs() - 256 * U * size)[~reached].max() <= 0


@pytest.mark.parametrize("held", [True, False])
def test_starts_that_reach_beyond_the_rows(held):
    """A batch cut short, or static starts: a row's place goes by the starts and not by the rows that are there."""
    for keep in (31, 17, 16, 3, 1):
        b = Batch([5, 0, 40], [20, 9, 30], 4, 2, 64, 16, torch.bfloat16, held, seed=keep)
        b.qkv = b.qkv[:keep]
        d = b.device()
        b.check(b.call(d), d)
    # single rows, and a sequence whose other rows are all missing
    b = Batch([15, 7, 3], [1, 1, 12], 4, 2, 64, 16, torch.float16, held, seed=1)
    b.qkv = b.qkv[:3]
    d = b.device()
    b.check(b.call(d), d)


def e4m3_borders():
    v = cache8.to_e4m3(torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16)
                                     for m in range(8)][:127], dtype=torch.float64))
    return (v[1:] + v[:-1]) / 2


@pytest.mark.parametrize("past,new,starts", [(9, 5, True), (30, 70, True), (3, 1, True), (40, 1, False)])
@pytest.mark.parametrize("scale", [0.3, 1.7e-3, 1.0, 0.25])
def test_keys_next_to_a_border_between_codes(scale, past, new, starts):
    """Keys that 64 bits tell from a border between two codes and 32 bits do not: angles of 24 bits are made so that a key of an
    8-bit number and an angle is the border times the scale, to half a step of 32 bits, on either side of it.  Scales of any
    value, as a user's cache may have them, are kept while they suffice."""
    D, BS, Hk = 64, 128, 2
    b = Batch([past], [new], 2, Hk, D, BS, torch.bfloat16, True, norm=None, spread=False, seed=new, starts=starts)
    b.ks[:], b.vs[:] = scale, scale
    border = e4m3_borders()
    border = border[(border > 2.0 ** -6) & (border < 250)]
    gen = torch.Generator().manual_seed(past)
    _, k, _ = b.parts(b.qkv)
    k[..., D // 2:] = 0
    rows = torch.arange(past, past + new)
    at = border[torch.randint(0, border.numel(), (new, D // 2), generator=gen)]
    low = torch.randint(128, 256, (new, D // 2), generator=gen).double()
    want = at * b.ks[0, 0].double()          # (the scale is fp32)
    low *= torch.exp2(torch.floor(torch.log2(want)) - 7)
    k[:, :, :D // 2] = low[:, None].to(torch.bfloat16) * torch.tensor([1.0, -1.0])[None, :, None].to(torch.bfloat16)
    b.cos[rows] = (want / low).float()
    b.sin[rows] = 0
    d = b.device()
    b.check(b.call(d), d)


@pytest.mark.parametrize("scale", [49 / 64, 99 / 512, 105.0, 0.5])
@pytest.mark.parametrize("new", [16, 60])
def test_values_on_a_border_between_codes(scale, new):
    """Values that are a border times the scale: the even one of the two codes.  (A product with the scale's reciprocal misses
    some of them, of scales that are no powers of two.)"""
    D, BS = 64, 128
    b = Batch([3], [new], 1, 1, D, BS, torch.float16, True, spread=False, seed=3)
    b.ks[:], b.vs[:] = 512.0, scale
    border = e4m3_borders()
    exact = border * scale
    exact = exact[(exact.to(torch.float16).double() == exact) & (exact < 448 * scale / 2)]
    assert exact.numel() > 30
    _, _, v = b.parts(b.qkv)
    v[:] = exact[torch.arange(new * D) % exact.numel()].view(new, 1, D).to(torch.float16)
    v[:, :, ::3] *= -1
    d = b.device()
    b.check(b.call(d), d)


@pytest.mark.parametrize("native", [True, False])
def test_eps_is_taken_in_64_bits(native, monkeypatch):
    """Normed keys next to borders between codes, by weights of 24 bits, with an eps that 32 bits change by half a step."""
    if not native:
        from flagattention_b200 import _native
        monkeypatch.setattr(_native, "usable", lambda x: False)
    D, BS, new = 64, 16, 16
    eps = 4.0 * (1 + 2.0 ** -24 - 2.0 ** -40)
    assert abs(float(torch.tensor(eps, dtype=torch.float32)) / eps - 1) > 2.0 ** -25
    b = Batch([0] * new, [1] * new, 1, 1, D, BS, torch.bfloat16, True, norm="fp32", spread=False, seed=1)
    border = e4m3_borders()
    border = border[(border >= 240) & (border < 448)]
    q, k, v = b.parts(b.qkv)
    k[:] = k[:1].clone()          # every sequence has one token, the same one at other positions: angles of 0
    b.cos[:], b.sin[:] = 1.0, 0.0
    x = k[0, 0].double()
    r = 1 / torch.sqrt((x * x).mean() + eps)
    at = border[torch.arange(D) % border.numel()] / 256.0
    b.wk = (at / (x * r)).float()
    lens, table, starts = b.lens, b.table, b.starts
    d = b.device()
    kc, vc = d["kc"].view(E4M3), d["vc"].view(E4M3)
    fa.rotary_and_cache(*b.parts(d["qkv"]), kc, vc, d["lens"], d["table"], d["cos"], d["sin"], query_starts=d["starts"],
                        q_weight=d["wq"], k_weight=d["wk"], eps=eps, key_scales=d["ks"], value_scales=d["vs"])
    want, ks = b.kc.view(E4M3).double(), b.ks.double()
    cache8.rotary_and_cache(q, k, v, want, b.vc.view(E4M3).double(), lens, table, b.cos, b.sin, starts, None, b.wq, b.wk, eps,
                            False, ks, b.vs.double())
    assert torch.equal(d["ks"].cpu().double(), ks)
    assert torch.equal(d["kc"].cpu().view(E4M3).double()[table[:, 0].long()], want[table[:, 0].long()])


@pytest.mark.parametrize("B,L,D", [(1, 1, 64), (3, 37, 96), (2, 9, 256)])
def test_eps_of_zero(B, L, D):
    """Lengths that leave places of the last strip of positions empty: those have no part in the weights' gradients."""
    gen = torch.Generator().manual_seed(L)
    q, g = (torch.randn(B, 3, L, D, generator=gen).to(torch.bfloat16) for _ in range(2))
    w = 1 + 0.3 * torch.randn(D, generator=gen)
    cos, sin = fa.rotary_tables(L, D)
    x, ws = q.cuda().requires_grad_(), w.cuda().requires_grad_()
    y, _ = fa.qk_norm_rotary(x, x.detach(), ws, w.cuda(), cos.cuda(), sin.cuda(), eps=0.0)
    dx, dw = torch.autograd.grad(y, (x, ws), g.cuda())
    want = cache8.norm_rotary(q, w, cos, sin, eps=0.0)
    size = torch.maximum(*(cache8.norm_rotary(q.abs(), w.abs(), cos.abs(), s, eps=0.0).abs() for s in (sin.abs(), -sin.abs())))
    dx64, dw64, dx_size, dw_size = cache8.norm_rotary_backward(q, w, g, cos, sin, eps=0.0)
    for got, want, half, terms, size in ((y, want, 2.0 ** -8, 64, size), (dx, dx64, 2.0 ** -8, 128, dx_size),
                                         (dw, dw64, 2.0 ** -24, 256, dw_size)):
        assert ((got.detach().cpu().double() - want).abs() <= half * want.abs() * (1 + half) + terms * U * size).all()


@pytest.mark.parametrize("exponent", [-112, -118, -126, -127, -131])
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("group", [2, 16])
def test_the_smallest_scales_of_values(exponent, splits, group):
    """bf16 holds 2^-126, and less in fewer bits, so scales down to there and below (codes are up to 448) are seen in the output.

    The bound of test_paged_8bit_gpu.py, and half of bf16's least step; fp32's own, 2^-149, once for each partition."""
    from test_paged_8bit_gpu import made
    x = made([700, 33, 16], 2 * group, 2, 128, 16, torch.bfloat16, seed=group)
    q, kc, vc, ks, vs, lens, bt = x
    last = vs[-1].clone()
    vs[:] = 2.0 ** exponent
    vs[1::3] = 1.25 * 2.0 ** (exponent + 1)
    vs[-1] = last
    out = fa.paged_attention_8bit(*(t.cuda() for t in x), 128 ** -0.5, 700, splits)
    want, size, most = cache8.paged_attention_8bit(*x, 128 ** -0.5)
    assert want.abs().max() > 2.0 ** exponent
    half = 2.0 ** -8
    bound = half * want.abs() * (1 + half) + (64 * 2.0 ** -23 * most + 2.0 ** -20 + 2.0 ** -17) * size + 2.0 ** -134 + 2.0 ** -147
    assert ((out.cpu().double() - want).abs() <= bound).all()


def test_small_scales_beside_large_ones_and_of_keys():
    """A scale below the normal numbers is a positive number like others: of a key, and of a value beside a larger one."""
    from test_paged_8bit_gpu import check, made
    x = made([200, 48], 8, 2, 64, 16, torch.float16, seed=4)
    q, kc, vc, ks, vs, lens, bt = x
    ks[:-1:2] = 2.0 ** -133
    vs[1:-1:3] = 2.0 ** -140
    check(fa.paged_attention_8bit(*(t.cuda() for t in x), 0.125, 200), x, 0.125)


@pytest.mark.parametrize("held", [True, False])
def test_chunks_behind_cached_tokens_attend_row_by_row(held):
    """Rows of prompts as sequences of their own, a length and a row of the table each, over what rotary_and_cache wrote.

    The bound of test_paged_8bit_gpu.py, and what the least numbers of fp16 cost, which the old codes here (any bits) show: a
    weight exp2(score - reference) s, s the scale (1 for 16 bits), goes in as an fp16 value, cut, and an fp16 remainder that
    is kept at 2^-24 or more (split_weights): off by 2^-24 where it is small, whatever the value beside it.  References are
    at most the largest score (and scale), 8-bit weights stand 2^6 above theirs: 2^-30 (16 bits: 2^-24) max(p s) sum |code|
    of the output, p the softmax."""
    b = Batch([20, 0, 33], [13, 40, 1], 8, 2, 64, 16, torch.float16, held, seed=5, spread=False)
    d = b.device()
    q = b.call(d)
    starts, lens = d["starts"].long(), d["lens"].long()
    rows = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(starts, rows, right=True) - 1
    row_lens = (lens[seq] - (starts[seq + 1] - 1 - rows)).to(torch.int32)
    table = d["table"][seq]
    assert row_lens.tolist() == list(range(21, 34)) + list(range(1, 41)) + [34]
    kc, vc, ks, vs = (d[n] for n in ("kc", "vc", "ks", "vs"))
    if held:
        kc, vc = kc.view(E4M3), vc.view(E4M3)
        o = fa.paged_attention_8bit(q, kc, vc, ks, vs, row_lens, table, 0.125, 40)
    else:
        ks = vs = torch.ones(kc.shape[:2], device="cuda")
        o = fa.paged_attention(q, kc, vc, row_lens, table, 0.125, 40)
    x = [t.cpu() for t in (q, kc, vc, ks, vs, row_lens, table)]
    want, size, most = cache8.paged_attention_8bit(*x, 0.125)
    q, kc, vc, ks, vs = (t.double() for t in x[:5])
    least = torch.zeros_like(want)
    for i, n in enumerate(row_lens.tolist()):
        ids = x[6][i].long()
        k, v = (c[ids].transpose(0, 1).flatten(1, 2)[:, :n] for c in (kc * ks[..., None, None], vc))
        s = vs[ids].t().repeat_interleave(16, 1)[:, :n]
        p = torch.softmax(q[i].view(2, 4, 64) @ k.transpose(1, 2) * 0.125, -1)
        top = (p * s[:, None]).amax(-1, keepdim=True)
        least[i] = (2.0 ** (-30 if held else -24) * top * v.abs().sum(1, keepdim=True)).flatten(0, 1)
    half = 2.0 ** -11
    bound = half * want.abs() * (1 + half) + (64 * 2.0 ** -23 * most + 2.0 ** -20 + 2.0 ** -17) * size + least + 2.0 ** -25
    assert o.isfinite().all() and ((o.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_weight_that_is_no_number_stays_in_its_column(interleaved):
    """Behind the rotated elements: one column of the queries and the keys, whatever the cache."""
    D, R = 128, 64
    for held in (True, False):
        b = Batch([3, 20], [18, 5], 2, 2, D, 16, torch.bfloat16, held, R=R, seed=1, interleaved=interleaved)
        b.wq[R + 3], b.wk[R + 9], b.wk[D - 1] = float("nan"), float("inf"), float("nan")
        d = b.device()
        out = b.call(d)
        want_q, kc, vc, ks, vs = b.expected()
        assert not same_where_not_finite(out, want_q)[:, :, R + 3].any()
        if held:
            got = d["kc"].cpu().view(E4M3).double()
            assert ((got == kc) | (got.isnan() & kc.isnan())).all() and torch.equal(d["ks"].cpu().double(), ks)
        else:
            same_where_not_finite(d["kc"], kc)
    q, w = torch.randn(1, 2, 9, D, device="cuda").half(), torch.ones(D, device="cuda")
    w[R + 3] = float("nan")
    y, _ = fa.qk_norm_rotary(q, q, w, w, *fa.rotary_tables(9, R, device="cuda"), interleaved=interleaved)
    bad = torch.zeros(D, dtype=torch.bool, device="cuda")
    bad[R + 3] = True
    assert torch.equal(y.isnan(), bad.expand_as(y))
