"""paged_attention_8bit against its definition in 64 bits.

Tolerance.  A score is a sum of at most 256 exact products in fp32, in the tensor cores' order: 32 x 2^-23 of the sum of
their sizes, times log2(e), is more than it loses, scaling included; it moves a weight by that times ln 2, in numerator
and denominator.  Weights go in as 22 bits and their exponentials are good to 2^-22: 2^-20 of sum |p v| bounds both, and
256 fp32 additions of up to 4096 tokens in runs of 128 and partial sums another 2^-17.  Then the output is rounded once."""
import pytest
import torch

import flagattention_b200 as fa
from oracle import cache8

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def made(lens, Hq, Hk, D, BS, dtype, seed=0, table=torch.int32, scales="powers", std=1.0, cols=None):
    gen = torch.Generator().manual_seed(seed)
    used = [-(-n // BS) for n in lens]
    NB = sum(used) + 2
    q = (torch.randn(len(lens), Hq, D, generator=gen) * std).to(dtype)
    codes = [torch.randn(NB, Hk, BS, D, generator=gen).mul(60).clamp(-448, 448).to(E4M3) for _ in range(2)]
    if scales == "powers":
        s = [torch.exp2(torch.randint(-8, -3, (NB, Hk), generator=gen).float()) for _ in range(2)]
    else:
        s = [torch.rand(NB, Hk, generator=gen) * 0.05 for _ in range(2)]
    order = torch.randperm(NB - 1, generator=gen)
    bt = torch.full((len(lens), cols or max(used + [1])), NB - 1, dtype=table)
    at = 0
    for i, n in enumerate(used):
        bt[i, :n] = order[at:at + n].to(table)
        at += n
    for c in codes:                      # what no table names, and what lies behind a sequence's end, must not matter
        c.view(torch.uint8)[NB - 1] = 127
    for i, n in enumerate(lens):
        if n % BS:
            for c in codes:
                c.view(torch.uint8)[int(bt[i, used[i] - 1]), :, n % BS:] = 127
    s[0][NB - 1] = s[1][NB - 1] = float("nan")
    return q, *codes, *s, torch.tensor(lens, dtype=torch.int32), bt


def call(x, scale, most, splits=0):
    q, kc, vc, ks, vs, lens, bt = (t.cuda() for t in x)
    return fa.paged_attention_8bit(q, kc, vc, ks, vs, lens, bt, scale, most, splits)


def check(out, x, scale, more=0.0):
    q, kc, vc, ks, vs, lens, bt = x
    want, size, most = cache8.paged_attention_8bit(q, kc, vc, ks, vs, lens, bt, scale)
    half = torch.finfo(q.dtype).eps / 2
    got = out.cpu().double()
    assert out.dtype == q.dtype and torch.isfinite(got).all()
    bound = half * want.abs() * (1 + half) + (2 * 32 * 2.0 ** -23 * most + 2.0 ** -20 + 2.0 ** -17 + more) * size
    off = (got - want).abs() - bound - (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    assert off.max() <= 0, f"over its bound by {off.max():.3e} of {want.abs().max():.3e}"


CASES = [
    # lens, Hq, Hk, D, BS, bound
    ([1], 1, 1, 16, 16, 1),
    ([0, 1, 15, 16, 17], 4, 2, 64, 16, 64),
    ([31, 32, 33, 300], 8, 8, 128, 16, 300),
    ([257, 1023, 5], 32, 8, 128, 16, 4096),
    ([700, 64, 129], 10, 1, 128, 64, 2000),
    ([1500, 1], 16, 1, 256, 32, 8192),
    ([333, 90], 40, 2, 64, 128, 333),
    ([2049], 7, 7, 32, 16, 32768),
    ([600, 601], 20, 1, 256, 16, 700),
    ([95, 96, 97], 6, 2, 128, 48, 200),
    ([3000] * 3 + [11], 64, 4, 128, 16, 4000),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_definition(case, dtype):
    lens, Hq, Hk, D, BS, most = CASES[case]
    x = made(lens, Hq, Hk, D, BS, dtype, seed=case, table=torch.int64 if case % 2 else torch.int32,
             scales="powers" if case % 3 else "any")
    check(call(x, D ** -0.5, most), x, D ** -0.5)


@pytest.mark.parametrize("splits", [1, 2, 5, 16])
@pytest.mark.parametrize("D,BS", [(128, 16), (64, 64), (256, 16)])
def test_given_split_counts(splits, D, BS):
    x = made([1000, 1, 63, 0, 640], 8, 2, D, BS, torch.float16, seed=splits)
    check(call(x, D ** -0.5, 1000, splits), x, D ** -0.5)


def test_many_sequences_sized_on_the_gpu():
    gen = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 700, (80,), generator=gen).tolist()
    x = made(lens, 8, 2, 128, 16, torch.bfloat16)
    for most in (700, 9000, 100000):
        check(call(x, 128 ** -0.5, most), x, 128 ** -0.5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scales_far_apart(dtype):
    """Blocks of very different scales, among them 0 and the least normal one: weights that no common 16-bit range holds."""
    x = made([400, 64], 8, 2, 128, 16, dtype, seed=5)
    vs, ks = x[4], x[3]
    vs[::3] *= 2.0 ** 20
    vs[1::5] = 0.0
    vs[2::7] = 2.0 ** -126
    ks[::4] = 0.0
    vs[-1] = float("nan")
    q = x[0]
    q.mul_(4)          # peaked
    if dtype == torch.float16:
        vs.clamp_(max=1.0)   # (what fp16 holds)
    check(call(x, 128 ** -0.5, 400), x, 128 ** -0.5)
    check(call(x, 128 ** -0.5, 400, 1), x, 128 ** -0.5)


def test_one_token_decides_in_a_block_of_tiny_values():
    """The softmax's maximum lies where V's scale is least: the output's reference and the sum's are far apart."""
    x = made([200], 4, 1, 64, 16, torch.bfloat16, seed=2)
    q, kc, vc, ks, vs, lens, bt = x
    b = int(bt[0, 7])
    vs[b] = 2.0 ** -100
    kc[b, 0, 3] = (q[0, 0].float() * 100).clamp(-448, 448).to(E4M3)
    check(call(x, 1.0, 200, 1), x, 1.0)
    check(call(x, 1.0, 200, 3), x, 1.0)


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 60])
def test_bf16_queries_of_any_size(scale):
    """Powers of two taken out of a row and put back into its scores: the same softmax as for rows of ordinary size."""
    x = made([100, 50], 4, 2, 64, 16, torch.bfloat16, seed=2)
    ref = call(x, 0.125, 100)
    y = (x[0] * scale, *x[1:])
    assert torch.equal(call(y, 0.125 / scale, 100), ref)


def test_strided_operands():
    """Queries as slices of a projection, caches as a layer of a pool or with heads inside tokens, tables with gaps."""
    x = made([77, 300], 8, 2, 64, 16, torch.float16, seed=3, cols=24)
    q, kc, vc, ks, vs, lens, bt = (t.cuda() for t in x)
    ref = fa.paged_attention_8bit(q, kc, vc, ks, vs, lens, bt, 0.125, 300)
    check(ref, x, 0.125)
    wide = torch.zeros(2, 12, 64, dtype=q.dtype, device="cuda")
    wide[:, 2:10] = q
    pools = []
    for c in (kc, vc):
        p = torch.zeros(c.shape[0], 3, *c.shape[1:], dtype=torch.uint8, device="cuda")
        p[:, 1] = c.view(torch.uint8)
        pools.append(p[:, 1].view(E4M3))
    tok = [c.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(E4M3) for c in (kc, vc)]
    wide_bt = torch.full((4, 40), -1, dtype=torch.int32, device="cuda")
    wide_bt[::2, :24] = bt
    for args in ((wide[:, 2:10], kc, vc, ks, vs, lens, bt), (q, *pools, ks, vs, lens, wide_bt[::2, :24]),
                 (q, *tok, ks, vs, lens.long(), bt.long()), (q.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, ks, vs, lens, bt),
                 (torch.cat((q[..., :3], q), -1)[..., 3:], kc, vc, ks, vs, lens, bt)):
        assert torch.equal(fa.paged_attention_8bit(*args, 0.125, 300), ref)


def test_a_cache_beyond_32_bits():
    """Blocks more than 2^32 codes into the cache."""
    D, Hk, BS = 128, 8, 16
    NB = (1 << 32) // (Hk * BS * D) + 40
    x = made([90, 33], 8, Hk, D, BS, torch.float16, seed=7)
    q, kc, vc, ks, vs, lens, bt = x
    n = kc.shape[0]
    big = []
    for c, s in ((kc, ks), (vc, vs)):
        cache = torch.empty(NB, Hk, BS, D, dtype=torch.uint8, device="cuda")
        sc = torch.empty(NB, Hk, device="cuda")
        cache[NB - n:] = c.view(torch.uint8).cuda()
        sc[NB - n:] = s.cuda()
        big += [cache.view(E4M3), sc]
    out = fa.paged_attention_8bit(q.cuda(), big[0], big[2], big[1], big[3], lens.cuda(), bt.cuda() + (NB - n), D ** -0.5, 90)
    check(out, x, D ** -0.5)


def test_tables_without_columns_and_no_sequences():
    x = [t.cuda() for t in made([40, 3], 4, 2, 64, 16, torch.float16)]
    assert (fa.paged_attention_8bit(*x[:6], x[6][:, :0], 0.125, 40) == 0).all()
    assert fa.paged_attention_8bit(x[0][:0], *x[1:5], x[5][:0], x[6][:0], 0.125, 40).shape == (0, 4, 64)
    x[5].fill_(-3)       # no length
    assert (fa.paged_attention_8bit(*x, 0.125, 40) == 0).all() and (fa.paged_attention_8bit(*x, 0.125, 9000) == 0).all()


def test_a_table_narrower_than_the_lengths():
    """Tokens without a column of the table are not there."""
    x = made([100, 64], 4, 2, 64, 16, torch.float16, seed=3)
    short = (*x[:6], x[6][:, :4].contiguous())
    same = (*x[:5], torch.tensor([64, 64], dtype=torch.int32), short[6])
    assert torch.equal(call(short, 0.125, 100, 1), call(same, 0.125, 100, 1))
    for most, splits in ((100, 2), (100, 0), (9000, 0)):
        check(call(short, 0.125, most, splits), same, 0.125)


@pytest.mark.parametrize("D,Hq,BS", [(128, 8, 16), (64, 8, 32), (128, 32, 48), (256, 2, 16), (16, 24, 64)])
@pytest.mark.parametrize("packed", [True, False])
def test_one_pass_over_long_sequences(D, Hq, BS, packed):
    """A warp's places are worked out 32 pieces at a time: around the ends of those, and an id that is wrong behind them.

    One pass: a warp adds its n / 64 pieces up, as value and remainder, in fp32 that the tensor cores may truncate, and
    their weights, two a piece and lane."""
    lens = [2047, 2048, 2049, 2064, 4095, 4097, 6150, 1]
    x = made(lens, Hq, 2, D, BS, torch.float16, seed=D + BS)
    q, kc, vc, ks, vs, n, bt = (t.cuda() for t in x)
    if not packed:   # heads inside tokens
        kc, vc = (c.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(E4M3) for c in (kc, vc))
    out = fa.paged_attention_8bit(q, kc, vc, ks, vs, n, bt, D ** -0.5, max(lens), 1)
    check(out, x, D ** -0.5, (2 * max(lens) / 64 + 4) * 2.0 ** -23 + 2 * max(lens) / 64 * 2.0 ** -24)
    bt[6, 6000 // BS] = kc.shape[0]
    bt[1, 0] = -5
    bad = fa.paged_attention_8bit(q, kc, vc, ks, vs, n, bt, D ** -0.5, max(lens), 1)
    good = [0, 2, 3, 4, 5, 7]
    assert torch.isnan(bad[[1, 6]]).all() and torch.equal(bad[good], out[good])


def test_ids_outside_the_cache_give_nan_and_nothing_else():
    x = made([100, 100, 40], 4, 2, 64, 16, torch.float16, seed=3)
    good = call(x, 0.125, 100)
    for bad in (-1, 10 ** 6):
        x[6][1, 2] = bad
        for splits in (0, 1, 2):
            out = call(x, 0.125, 100, splits)
            assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2]]).all()
    assert torch.equal(call(x, 0.125, 100)[[0, 2]], good[[0, 2]])


def test_nan_codes_of_visible_tokens_show():
    x = made([100, 100], 4, 2, 64, 16, torch.float16, seed=3)
    x[1].view(torch.uint8)[int(x[6][0, 1]), 0, 3, 7] = 127
    out = call(x, 0.125, 100)
    assert torch.isnan(out[0, :2]).all() and torch.isfinite(out[0, 2:]).all() and torch.isfinite(out[1]).all()


def test_captured_step_follows_lengths_on_a_side_stream():
    x = made([300, 77], 8, 2, 128, 16, torch.bfloat16, seed=3)
    d = [t.cuda() for t in x]
    most = 5000
    want = []
    steps = ([300, 77], [12, 0], [1, 77])
    for s in steps:
        d[5].copy_(torch.tensor(s))
        want.append(fa.paged_attention_8bit(*d, 0.1, most))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = fa.paged_attention_8bit(*d, 0.1, most)
    for s, w in zip(steps, want):
        d[5].copy_(torch.tensor(s))
        graph.replay()
        assert torch.equal(out, w)


def test_same_codes_as_the_16_bit_cache():
    """Over a 16-bit cache that holds the very values, paged_attention gives the same within both roundings."""
    x = made([500, 31, 250], 16, 4, 128, 16, torch.float16, seed=4, scales="powers")
    q, kc, vc, ks, vs, lens, bt = (t.cuda() for t in x)
    k16, v16 = ((c.float() * s[..., None, None]).half() for c, s in ((kc, ks), (vc, vs)))
    a = fa.paged_attention_8bit(q, kc, vc, ks, vs, lens, bt, 128 ** -0.5, 500).float()
    b = fa.paged_attention(q, k16, v16, lens, bt, 128 ** -0.5, 500).float()
    size = cache8.paged_attention_8bit(*x, 128 ** -0.5)[1].cuda()
    assert ((a - b).abs() <= 2 * 2.0 ** -11 * b.abs() + 2.0 ** -12 * size).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_run_of_prompts_and_steps(dtype):
    """Prompts written at once, then three decode steps of append and attention, against the same run in 64 bits."""
    gen = torch.Generator().manual_seed(9)
    Hq, Hk, D, BS, lens = 8, 2, 128, 16, [37, 200, 16, 1]
    S, cols = len(lens), 14
    bt = torch.randperm(S * cols, generator=gen).view(S, cols).to(torch.int32)
    cos, sin = fa.rotary_tables(300, D)
    wq, wk = (1 + 0.2 * torch.randn(D, generator=gen) for _ in range(2))
    kc, vc = (torch.zeros(S * cols, Hk, BS, D, dtype=E4M3, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(S * cols, Hk, device="cuda") for _ in range(2))
    ref = [torch.zeros(S * cols, Hk, BS, D, dtype=torch.float64) for _ in range(2)] + \
        [torch.zeros(S * cols, Hk, dtype=torch.float64) for _ in range(2)]
    now = torch.tensor(lens, dtype=torch.int32)
    for step in range(4):
        T = sum(lens) if step == 0 else S
        q, k, v = (torch.randn(T, h, D, generator=gen).to(dtype) for h in (Hq, Hk, Hk))
        starts = torch.tensor([0] + lens).cumsum(0) if step == 0 else None
        if step:
            now = now + 1
        out = fa.rotary_and_cache(q.cuda(), k.cuda(), v.cuda(), kc, vc, now.cuda(), bt.cuda(), cos.cuda(), sin.cuda(),
                                  query_starts=None if starts is None else starts.cuda(), q_weight=wq.cuda(),
                                  k_weight=wk.cuda(), key_scales=ks, value_scales=vs)
        cache8.rotary_and_cache(q, k, v, ref[0], ref[1], now, bt, cos, sin, starts, None, wq, wk, key_scales=ref[2],
                                value_scales=ref[3])
        assert torch.equal(kc.cpu().double(), ref[0]) and torch.equal(vc.cpu().double(), ref[1])
        assert torch.equal(ks.cpu().double(), ref[2]) and torch.equal(vs.cpu().double(), ref[3])
        if step:
            o = fa.paged_attention_8bit(out, kc, vc, ks, vs, now.cuda(), bt.cuda(), D ** -0.5, 400)
            check(o, (out.cpu(), ref[0], ref[1], ref[2], ref[3], now, bt), D ** -0.5)
