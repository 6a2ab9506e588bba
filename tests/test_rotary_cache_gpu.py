"""rotary_and_cache against its definition in 64 bits.  Codes of 8 bits and their scales are equal to the last bit: the
kernel works them out in 64 bits and rounds once.  Queries, and keys of a 16-bit cache, are fp32 arithmetic rounded once:
half a step of the type and 64 fp32 roundings of the terms' sizes (as in test_qk_norm_gpu.py)."""
import pytest
import torch

import flagattention_b200 as fa
from oracle import cache8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
E4M3 = torch.float8_e4m3fn


class Batch:
    """Sequences with tokens in a cache and new ones, on the CPU, and their copies on the GPU."""

    def __init__(self, past, new, Hq, Hk, D, BS, dtype, held, R=None, norm="fp32", interleaved=False, starts=True, pad=0,
                 seed=0, table=torch.int32, cols=None, spread=True):
        gen = torch.Generator().manual_seed(seed)
        self.gen, self.held, self.dtype, self.BS = gen, held, dtype, BS
        T = sum(new) + pad
        qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=gen)
        if spread:
            qkv *= torch.exp2(torch.randint(-4, 5, (T, 1), generator=gen).float())
        self.qkv = qkv.to(dtype)
        self.heads = (Hq, Hk, D)
        lens = [p + n for p, n in zip(past, new)]
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.starts = torch.tensor([0] + new).cumsum(0).to(torch.int32) if starts else None
        used = [-(-n // BS) for n in lens]
        self.NB = sum(used) + 3
        order = torch.randperm(self.NB, generator=gen)
        self.table = torch.full((len(new), cols or max(used + [1])), -1, dtype=table)
        at = 0
        for i, n in enumerate(used):
            self.table[i, :n] = order[at:at + n].to(table)
            at += n
        shape = (self.NB, Hk, BS, D)
        if held:
            self.kc, self.vc = (torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8) for _ in range(2))
            for c in (self.kc, self.vc):
                c[(c & 127) == 127] = 0          # (no NaN among the old codes)
            self.ks, self.vs = (torch.exp2(torch.randint(-9, 2, shape[:2], generator=gen).float()) for _ in range(2))
        else:
            self.kc, self.vc = (torch.randn(shape, generator=gen).to(dtype) for _ in range(2))
            self.ks = self.vs = None
        wtype = torch.float32 if norm == "fp32" else dtype
        self.wq, self.wk = ((1 + 0.3 * torch.randn(D, generator=gen)).to(wtype) for _ in range(2)) if norm else (None, None)
        self.cos, self.sin = fa.rotary_tables(max(lens + [1]) + 1, R or D)
        self.interleaved, self.positions = interleaved, None

    def parts(self, qkv):
        Hq, Hk, D = self.heads
        x = qkv.view(qkv.shape[0], Hq + 2 * Hk, D)
        return x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]

    def device(self):
        return {n: None if getattr(self, n) is None else getattr(self, n).cuda()
                for n in ("qkv", "lens", "starts", "table", "kc", "vc", "ks", "vs", "wq", "wk", "cos", "sin", "positions")}

    def call(self, d):
        kc, vc = (d["kc"].view(E4M3), d["vc"].view(E4M3)) if self.held else (d["kc"], d["vc"])
        return fa.rotary_and_cache(*self.parts(d["qkv"]), kc, vc, d["lens"], d["table"], d["cos"], d["sin"],
                                   query_starts=d["starts"], positions=d["positions"], q_weight=d["wq"], k_weight=d["wk"],
                                   interleaved=self.interleaved, key_scales=d["ks"], value_scales=d["vs"])

    def expected(self, abs_=False):
        """(queries, key cache, value cache, key scales, value scales) in 64 bits."""
        kc, vc = ((c.view(E4M3) if self.held else c).double() for c in (self.kc, self.vc))
        ks, vs = (None if s is None else s.double() for s in (self.ks, self.vs))
        q, k, v = self.parts(self.qkv.abs() if abs_ else self.qkv)
        sin = -self.sin.abs() if abs_ else self.sin
        cos = self.cos.abs() if abs_ else self.cos
        w = [None if t is None else t.abs() if abs_ else t for t in (self.wq, self.wk)]
        args = (self.lens, self.table, cos, sin, self.starts, self.positions, *w, 1e-6, self.interleaved)
        if not abs_:
            return (cache8.rotary_and_cache(q, k, v, kc, vc, *args, ks, vs), kc, vc, ks, vs)
        # the sum of the terms' sizes is in one of the two elements of a pair, for either sign of the sine
        sizes = []
        for s in (sin, -sin):
            kk = torch.zeros_like(kc)
            qq = cache8.rotary_and_cache(q, k, v, kk, torch.zeros_like(vc), *args[:3], s, *args[4:])
            sizes.append((qq.abs(), kk.abs()))
        return sizes[0][0].maximum(sizes[1][0]), sizes[0][1].maximum(sizes[1][1])

    def check(self, out, d):
        q, kc, vc, ks, vs = self.expected()
        q_size, k_size = self.expected(abs_=True)
        half, least = torch.finfo(self.dtype).eps / 2, 2.0 ** -25

        def near(got, want, size):
            off = (got.cpu().double() - want).abs() - half * want.abs() * (1 + half) - 64 * U * size
            return off.max() <= (least if self.dtype == torch.float16 else 0.0) if off.numel() else True

        assert out.dtype == self.dtype and near(out, q, q_size), "queries"
        if self.held:
            for name, got, want in (("key scales", d["ks"], ks), ("value scales", d["vs"], vs)):
                assert torch.equal(got.cpu().double(), want), name
            for name, got, want in (("keys", d["kc"], kc), ("values", d["vc"], vc)):
                got = got.cpu().view(E4M3).double()
                same = (got == want) | (got.isnan() & want.isnan())
                assert same.all(), f"{name}: {(~same).sum()} of {same.numel()} codes differ"
        else:
            assert torch.equal(d["vc"].cpu().double(), vc), "values"
            assert near(d["kc"], kc, k_size), "keys"


CASES = [
    # past, new, Hq, Hk, D, BS, extra
    ([0], [1], 1, 1, 16, 16, {}),
    ([15, 16, 31, 0], [1, 1, 1, 1], 4, 2, 64, 16, dict(starts=False)),
    ([5, 0, 17, 40], [30, 1, 16, 100], 8, 2, 128, 16, {}),
    ([7, 100, 0], [200, 3, 129], 5, 1, 128, 64, dict(interleaved=True, R=64)),
    ([0, 127, 60], [300, 2, 200], 3, 3, 256, 128, dict(pad=9)),
    ([1, 2, 3], [64, 31, 1], 4, 4, 32, 32, dict(R=16, norm=None)),
    ([3] * 70, [1] * 70, 16, 8, 128, 16, dict(norm="own", table=torch.int64)),
    ([0, 9, 0, 3, 0], [5, 0, 0, 40, 0], 2, 1, 64, 48, dict(pad=3)),
]


@pytest.mark.parametrize("held", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_definition(case, dtype, held):
    past, new, Hq, Hk, D, BS, extra = CASES[case]
    b = Batch(past, new, Hq, Hk, D, BS, dtype, held, seed=case, **extra)
    d = b.device()
    b.check(b.call(d), d)


@pytest.mark.parametrize("held", [True, False])
def test_many_sequences_and_mixed_batch(held):
    """More than 32 sequences (the search over query_starts goes round), empty ones, decode rows between prompts."""
    gen = torch.Generator().manual_seed(4)
    new = [1] * 40 + [0, 0, 50, 0] + [1] * 20 + [7, 33, 0]
    past = torch.randint(0, 90, (len(new),), generator=gen).tolist()
    b = Batch(past, new, 4, 2, 64, 16, torch.bfloat16, held, seed=9, pad=21)
    d = b.device()
    b.check(b.call(d), d)


@pytest.mark.parametrize("held", [True, False])
def test_rows_without_a_place(held):
    """Idle slots (length 0), more rows than tokens, a table too narrow, ids outside the cache: nothing is written, the
    queries are 0 (but where only the key has no block)."""
    b = Batch([3, 0, 20, 5], [4, 6, 1, 9], 2, 1, 64, 16, torch.float16, held, seed=2, cols=2)
    b.lens[1] = 4          # two rows in front of the sequence
    b.lens[0] = 0          # none has a place
    b.lens[2] = 40         # behind the table's two columns
    b.table[3, 0] = b.NB   # no such block
    d = b.device()
    b.check(b.call(d), d)
    b = Batch([3, 3, 3], [1, 1, 1], 2, 1, 64, 16, torch.float16, held, seed=2, starts=False)
    b.lens[1], b.table[2, 0] = 0, -7
    d = b.device()
    b.check(b.call(d), d)


@pytest.mark.parametrize("D,BS", [(128, 16), (64, 32), (256, 128)])
def test_token_by_token_is_all_at_once(D, BS):
    """A block filled in steps, scales growing, equals the block filled at once, but for codes that were below 2^-6 of the
    final scale (which e4m3 rounds twice)."""
    n = 2 * BS + 5
    whole = Batch([0], [n], 2, 2, D, BS, torch.bfloat16, True, seed=1)
    grow = torch.exp2(torch.arange(n).float() % BS / BS * 6)[:, None]
    whole.qkv = (whole.qkv.float() * grow).to(torch.bfloat16)
    d = whole.device()
    out = whole.call(d)
    e = whole.device()
    rows = []
    for i in range(n):
        one = {**e, "qkv": e["qkv"][i:i + 1], "lens": torch.tensor([i + 1], dtype=torch.int32, device="cuda"), "starts": None}
        rows.append(whole.call(one))
    assert torch.equal(torch.cat(rows), out)
    blocks = whole.table[0].long().cuda()
    for c, s in (("kc", "ks"), ("vc", "vs")):
        assert torch.equal(d[s][blocks], e[s][blocks])
        x, y = (t[c][blocks].view(E4M3).float().transpose(1, 2).flatten(0, 1)[:n] for t in (d, e))
        assert torch.equal(x[x.abs() >= 2.0 ** -6], y[x.abs() >= 2.0 ** -6])
        # below, moves lose half a step of 2^-9 each, of which half survives the next, and the one rounding of x as much:
        # less than a step and a half between two numbers that are whole steps
        assert ((x - y).abs() <= 2.0 ** -9).all()


def test_scales_that_the_user_made_grow_right():
    """Old scales that are no powers of two are kept while they suffice, and left behind when they do not."""
    b = Batch([9, 9], [2, 2], 1, 1, 64, 16, torch.bfloat16, True, seed=3, starts=True, spread=False)
    b.ks[:], b.vs[:] = 0.3, 0.0007
    d = b.device()
    b.check(b.call(d), d)


def test_values_that_no_scale_holds():
    """Infinities saturate, NaN stays, neither moves the scale; zeros and subnormals have the least scale."""
    b = Batch([0, 0, 0], [16, 16, 3], 1, 1, 64, 16, torch.bfloat16, True, seed=3, norm=None)
    q, k, v = b.parts(b.qkv)
    v[3, 0, 5], v[4, 0, 6], v[5, 0, 7] = float("inf"), -float("inf"), float("nan")
    v[16:32] = 0
    v[32:] = 1e-39
    k[20, 0, 1] = float("nan")
    d = b.device()
    b.check(b.call(d), d)


def test_positions_given():
    b = Batch([5, 30], [20, 7], 2, 1, 64, 16, torch.bfloat16, True, seed=3)
    b.positions = torch.randint(-4, 80, (27,), generator=b.gen)
    d = b.device()
    b.check(b.call(d), d)


def test_cache_views_and_other_strides():
    """Caches as slices of a larger pool (layers side by side), operands not aligned or not contiguous inside."""
    b = Batch([5, 30], [20, 7], 4, 2, 64, 16, torch.bfloat16, True, seed=3)
    d = b.device()
    for name in ("kc", "vc"):
        pool = torch.zeros(b.NB, 3, 2, 16, 64, dtype=torch.uint8, device="cuda")
        pool[:, 1] = d[name]
        d[name], d[name + "_pool"] = pool[:, 1], pool
    wide = torch.zeros(27, d["qkv"].shape[1] + 3, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:] = d["qkv"]
    x = wide[:, 3:].unflatten(1, (8, 64))
    kc, vc = d["kc"].view(E4M3), d["vc"].view(E4M3)
    out = fa.rotary_and_cache(x[:, :4], x[:, 4:6], x[:, 6:], kc, vc, d["lens"], d["table"], d["cos"], d["sin"],
                              query_starts=d["starts"].long(), q_weight=d["wq"], k_weight=d["wk"], key_scales=d["ks"],
                              value_scales=d["vs"])
    b.check(out, d)
    for name in ("kc", "vc"):
        assert (d[name + "_pool"][:, 0] == 0).all() and (d[name + "_pool"][:, 2] == 0).all()


def test_empty_call():
    b = Batch([5, 30], [0, 0], 4, 2, 64, 16, torch.bfloat16, True, seed=3)
    d = b.device()
    assert b.call(d).shape == (0, 4, 64)
    b.check(b.call(d), d)


@pytest.mark.parametrize("held", [True, False])
def test_rows_without_sequences_or_tables(held):
    """No sequence at all, and tables without a column: queries of 0, caches as they were."""
    b = Batch([], [], 4, 2, 64, 16, torch.bfloat16, held, seed=3, pad=7)
    d = b.device()
    assert d["lens"].numel() == 0
    out = b.call(d)
    assert out.shape == (7, 4, 64) and (out == 0).all()
    b = Batch([0, 0], [1, 1], 4, 2, 64, 16, torch.bfloat16, held, seed=3)
    b.table = b.table[:, :0]
    d = b.device()
    assert (b.call(d) == 0).all()
    assert torch.equal(d["kc"].cpu(), b.kc)
    b = Batch([3, 9], [4, 2], 4, 2, 64, 16, torch.bfloat16, held, seed=3)
    b.starts += 5        # rows in front of the first sequence
    b.qkv = torch.cat((b.qkv[:5], b.qkv))
    d = b.device()
    b.check(b.call(d), d)


def test_captured_step_follows_lengths():
    b = Batch([15, 3, 40], [1, 1, 1], 4, 2, 128, 16, torch.bfloat16, True, seed=6, starts=False, cols=5)
    b.cos, b.sin = fa.rotary_tables(100, 128)
    for i in range(3):     # room for the steps to come
        b.table[i] = torch.arange(5 * i, 5 * i + 5)
    b.NB = 15
    b.kc, b.vc, b.ks, b.vs = (t[:1].expand(15, *t.shape[1:]).clone() for t in (b.kc, b.vc, b.ks, b.vs))
    d, e = b.device(), b.device()
    want = []
    for step in range(3):
        e["lens"].copy_(b.lens + step)
        e["qkv"].copy_(b.qkv.cuda() * (step + 1))
        want.append(b.call(e).clone())
    b.call(d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.call(d)
    d.update({n: v for n, v in d.items()})
    for n in ("kc", "vc", "ks", "vs"):
        d[n].copy_(getattr(b, n))
    for step in range(3):
        d["lens"].copy_(b.lens + step)
        d["qkv"].copy_(b.qkv.cuda() * (step + 1))
        graph.replay()
        assert torch.equal(out, want[step])
    for n in ("kc", "vc", "ks", "vs"):
        assert torch.equal(d[n], e[n])
