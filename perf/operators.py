"""The work of the operators around attention in a decoder: norm and rotation of queries and keys, writing the paged
cache, and decoding over a cache held in 8 bits.

`listed()` names twelve calls, `draw()` gives more of the same ranges.  A case is a dict of plain values with an "op":

  norm_rotary  qk_norm_rotary: RMS norm of every head of q and k and the rotation by position, in (batch, heads,
               length, head_dim); with `grad` forward and backward to q, k and both weights
  append       rotary_and_cache: the new tokens of a batch of sequences, normed and rotated, into the paged caches, of
               16 bits or (`cache` = "e4m3") of 8 with a scale for each block and kv head
  decode       paged_attention_8bit: one query token a sequence over such a cache

`run()` computes them with elementary torch operations, or, where `own` is true, calls the operators.  Lengths are a
part of the case, so that every seed costs the same; the seed makes the values, the order of the blocks and the scales.
Activations are N(0, 1) with a few channels ten times as large, as queries and keys of trained models have them.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn
_LEAST = -126   # exponent of the least scale: the smallest normal fp32 number


def listed():
    return [
        # one step's tokens of a batch of requests before attention: the smallest call, latency
        dict(name="norm_rotary_token", op="norm_rotary", dtype="bf16", weights="bf16", B=16, H=32, Hk=8, L=1, D=128,
             R=128, interleaved=False, positions=True, layout="blhd", grad=False),
        # a training step of a grouped-query layer at the benchmark's length, master weights in 32 bits
        dict(name="norm_rotary_train", op="norm_rotary", dtype="bf16", weights="fp32", B=2, H=32, Hk=8, L=4096, D=128,
             R=128, interleaved=False, positions=False, layout="bhld", grad=True),
        # the same on sequences of no round length, half of a smaller head rotated in pairs of neighbours, q and k as
        # the projections leave them
        dict(name="norm_rotary_ragged", op="norm_rotary", dtype="fp16", weights="fp16", B=3, H=20, Hk=4, L=1999, D=64,
             R=32, interleaved=True, positions=False, layout="blhd", grad=True),
        # a long prompt of one request, its positions given
        dict(name="norm_rotary_long", op="norm_rotary", dtype="bf16", weights="bf16", B=2, H=48, Hk=8, L=16384, D=128,
             R=128, interleaved=False, positions=True, layout="blhd", grad=False),
        # a decode step's new tokens into a cache of 8 bits, some of them the first of their block
        dict(name="append8_decode", op="append", dtype="bf16", cache="e4m3", seqs=64, H=32, Hk=8, D=128, R=128, block=16,
             new_lo=1, new_hi=1, past_lo=1, past_hi=700, pad=0, norm=True, interleaved=False),
        # prompts of several requests packed into one call, 8 bits
        dict(name="append8_prompts", op="append", dtype="bf16", cache="e4m3", seqs=7, H=32, Hk=8, D=128, R=128, block=16,
             new_lo=300, new_hi=2100, past_lo=0, past_hi=400, pad=61, norm=True, interleaved=False),
        # a few requests' new tokens into a 16-bit cache, no norm
        dict(name="append16_decode", op="append", dtype="fp16", cache="16", seqs=5, H=16, Hk=2, D=64, R=64, block=16,
             new_lo=1, new_hi=1, past_lo=1, past_hi=2000, pad=0, norm=False, interleaved=True),
        # decode tokens and chunks of prompts in one call, 16-bit cache of larger blocks
        dict(name="append16_mixed", op="append", dtype="bf16", cache="16", seqs=33, H=28, Hk=4, D=128, R=64, block=32,
             new_lo=1, new_hi=999, past_lo=0, past_hi=1500, pad=17, norm=True, interleaved=False),
        # decoding for a full batch over a cache of 8 bits, lengths as in the benchmark of the 16-bit cache
        dict(name="decode8_batch", op="decode", dtype="fp16", seqs=64, H=32, Hk=8, D=128, block=16, lo=1024, hi=32768,
             most=32768, table="int32"),
        # a few short requests under a large bound: the smallest step of a serving loop
        dict(name="decode8_few", op="decode", dtype="bf16", seqs=4, H=32, Hk=8, D=128, block=16, lo=1, hi=1500,
             most=32768, table="int32"),
        # many requests of ordinary length, 16 query heads a kv head, larger blocks
        dict(name="decode8_ragged", op="decode", dtype="bf16", seqs=37, H=32, Hk=2, D=64, block=64, lo=1, hi=8191,
             most=8192, table="int64"),
        # one long document
        dict(name="decode8_one", op="decode", dtype="fp16", seqs=1, H=64, Hk=8, D=128, block=32, lo=131071, hi=131071,
             most=131072, table="int32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rotary", "append", "decode"])
    dtype = rng.choice(["bf16", "fp16"])
    Hk = rng.choice([1, 2, 3, 4, 5, 8])
    G = rng.choice([1, 2, 4, 5, 7, 8, 16])
    D = rng.choice([64, 128, 128, 256])
    if op == "norm_rotary":
        B, D = _log(rng, 1, 16), rng.choice([64, 80, 96, 128, 128, 192, 256])
        grad = rng.random() < 0.6
        H, L = Hk * G, 1 if rng.random() < 0.2 else _log(rng, 2, 8192)
        while B * L * (H + Hk) * D > (1 << 27):
            L = max(1, L // 2)
        return dict(op=op, dtype=dtype, weights=rng.choice([dtype, "fp32"]), B=B, H=H, Hk=Hk, L=L, D=D,
                    R=rng.choice([D, D, D // 32 * 16]), interleaved=rng.random() < 0.4, positions=rng.random() < 0.4,
                    layout=rng.choice(["bhld", "blhd"]), grad=grad)
    if op == "append":
        seqs, one = _log(rng, 1, 128), rng.random() < 0.4
        new = 1 if one else _log(rng, 2, 2048)
        while seqs * new * (Hk * G + 2 * Hk) * D > (1 << 26):
            new = max(1, new // 2)
        return dict(op=op, dtype=dtype, cache=rng.choice(["e4m3", "e4m3", "16"]), seqs=seqs, H=Hk * G, Hk=Hk, D=D,
                    R=rng.choice([D, D, D // 2]), block=rng.choice([16, 16, 32, 64, 128]), new_lo=1, new_hi=new,
                    past_lo=rng.choice([0, 1]), past_hi=_log(rng, 1, 2000), pad=0 if new == 1 else rng.choice([0, 5, 100]),
                    norm=rng.random() < 0.6, interleaved=rng.random() < 0.3)
    seqs, hi = _log(rng, 1, 64), _log(rng, 1, 65536)
    while seqs * hi * Hk * D > (1 << 30):
        hi = hi // 2
    return dict(op=op, dtype=dtype, seqs=seqs, H=Hk * G, Hk=Hk, D=D, block=rng.choice([16, 16, 32, 64, 128]),
                lo=rng.choice([0, 1, max(1, hi // 2)]), hi=hi, most=hi if rng.random() < 0.5 else hi + _log(rng, 1, 20000),
                table=rng.choice(["int32", "int64"]))


# ---- what a case holds -------------------------------------------------------------------------------------------------
def _lengths(case):
    """append: (cached before, new) of every sequence; decode: the context lengths."""
    rng = random.Random("%s %d %d" % (case["op"], case["seqs"], case["block"]))
    n = case["seqs"]
    if case["op"] == "append":
        return ([rng.randint(case["past_lo"], case["past_hi"]) for _ in range(n)],
                [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(n)])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(n)]


def _cdiv(a, b):
    return -(-a // b)


def work(case):
    if case["op"] == "norm_rotary":
        n, rows = case["B"] * case["L"], case["B"] * case["L"] * (case["H"] + case["Hk"])
        el, w = rows * case["D"], 2 * case["D"] * (4 if case["weights"] == "fp32" else 2)
        tables = (n if case["positions"] else case["L"]) * case["R"] * 4
        if not case["grad"]:
            return {"bytes": 4 * el + w + tables, "flops": 8 * el}
        return {"bytes": 10 * el + 2 * w + tables, "flops": 26 * el}
    if case["op"] == "append":
        past, new = _lengths(case)
        n, held = sum(new), 1 if case["cache"] == "e4m3" else 2
        units = sum(_cdiv(p + m, case["block"]) - p // case["block"] for p, m in zip(past, new))
        per = case["H"] * 4 + case["Hk"] * (4 + 2 * held)
        scales = units * case["Hk"] * 8 if held == 1 else 0
        return {"bytes": n * (per * case["D"] + case["R"] * 4) + scales + units * 4,
                "flops": 8 * n * (case["H"] + case["Hk"]) * case["D"]}
    lens = _lengths(case)
    blocks = sum(_cdiv(n, case["block"]) for n in lens)
    entry = 8 if case["table"] == "int64" else 4
    return {"bytes": sum(lens) * case["Hk"] * case["D"] * 2 + blocks * (case["Hk"] * 8 + entry)
            + case["seqs"] * (case["H"] * case["D"] * 4 + 4),
            "flops": 4 * sum(lens) * case["H"] * case["D"]}


def _activations(gen, shape, dtype):
    x = torch.randn(shape, generator=gen, device="cuda")
    x[..., 5::24] *= 10.0   # the channels that stand out
    return x.to(dtype)


def _tables(rows, R):
    """cos, sin (rows, R / 2) in 32 bits, the angles in 64."""
    freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def _weight(gen, D, dtype):
    return (1.0 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(dtype)


def _filled(gen, blocks, Hk, BS, D):
    """A cache of 8 bits with its scales, powers of two as the writer leaves them, of values N(0, 1) in blocks of
    different size: (codes, scales)."""
    codes = torch.empty(blocks, Hk, BS, D, dtype=_E4M3, device="cuda")
    scales = torch.empty(blocks, Hk, device="cuda")
    step = max(1, (1 << 26) // (Hk * BS * D))
    for i in range(0, blocks, step):   # a part of the cache at a time: the values need four times its room
        x = torch.randn(min(step, blocks - i), Hk, BS, D, generator=gen, device="cuda")
        x *= torch.exp2(torch.randint(-2, 3, x.shape[:2], generator=gen, device="cuda").float())[..., None, None]
        s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448.0)))
        codes[i:i + step] = (x / s[..., None, None]).to(_E4M3)
        scales[i:i + step] = s
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype, D, H, Hk = _DTYPES[case["dtype"]], case["D"], case["H"], case["Hk"]
    s = dict(case=dict(case))
    if case["op"] == "norm_rotary":
        B, L = case["B"], case["L"]

        def made(h):
            if case["layout"] == "bhld":
                return _activations(gen, (B, h, L, D), dtype)
            return _activations(gen, (B, L, h, D), dtype).transpose(1, 2)

        s.update(q=made(H), k=made(Hk), wq=_weight(gen, D, _DTYPES[case["weights"]]),
                 wk=_weight(gen, D, _DTYPES[case["weights"]]))
        rows = L
        s["positions"] = None
        if case["positions"]:   # requests that are at different places of their sequences
            rows = L + 4000
            s["positions"] = torch.randint(0, 4000, (B, 1), generator=gen, device="cuda") + torch.arange(L, device="cuda")
        s["cos"], s["sin"] = _tables(rows, case["R"])
        if case["grad"]:
            for name in ("q", "k", "wq", "wk"):
                s[name].requires_grad_()
            s["gq"], s["gk"] = (torch.randn(B, h, L, D, generator=gen, device="cuda").to(dtype) for h in (H, Hk))
        return s
    BS = case["block"]
    if case["op"] == "append":
        past, new = _lengths(case)
        total = sum(new) + case["pad"]
        # one projection gives query, key and value of a token side by side
        qkv = _activations(gen, (total, (H + 2 * Hk) * D), dtype).view(total, H + 2 * Hk, D)
        s.update(q=qkv[:, :H], k=qkv[:, H:H + Hk], v=qkv[:, H + Hk:])
        lens = [p + n for p, n in zip(past, new)]
        s["wq"], s["wk"] = (_weight(gen, D, dtype), _weight(gen, D, dtype)) if case["norm"] else (None, None)
        s["cos"], s["sin"] = _tables(max(lens) + 1, case["R"])
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["starts"] = None
        if case["pad"] or case["new_hi"] > 1:
            s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    else:
        lens = _lengths(case)
        s["q"] = _activations(gen, (case["seqs"], H, D), dtype)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # the pool's blocks in any order; the last one is not used, and unused entries of the table name it
    used = [_cdiv(n, BS) for n in lens]
    blocks = sum(used) + 1
    order = torch.randperm(blocks - 1, generator=gen, device="cuda")
    most = case.get("most", max(max(lens), 1))
    at = torch.arange(_cdiv(most, BS), device="cuda")[None]
    first = torch.tensor([0] + used, device="cuda").cumsum(0)[:-1, None]
    inside = at < torch.tensor(used, device="cuda")[:, None]
    table = torch.full(inside.shape, blocks - 1, device="cuda")
    table[inside] = order[(first + at)[inside]]
    s["table"] = table.to(torch.int64 if case.get("table") == "int64" else torch.int32)
    if case["op"] == "append" and case["cache"] == "16":
        s["kc"], s["vc"] = (torch.randn(blocks, Hk, BS, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
        s["ks"] = s["vs"] = None
    else:
        s["kc"], s["ks"] = _filled(gen, blocks, Hk, BS, D)
        s["vc"], s["vs"] = _filled(gen, blocks, Hk, BS, D)
    return s


# ---- the operators as a user calls them --------------------------------------------------------------------------------
def _own(s):
    import flagattention_b200 as fa
    case = s["case"]
    if case["op"] == "norm_rotary":
        q, k = fa.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"],
                                 case["interleaved"])
        if not case["grad"]:
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if case["op"] == "append":
        q = fa.rotary_and_cache(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["lens"], s["table"], s["cos"], s["sin"],
                                query_starts=s["starts"], q_weight=s["wq"], k_weight=s["wk"],
                                interleaved=case["interleaved"], key_scales=s["ks"], value_scales=s["vs"])
        return _appended(s, q)
    return {"o": fa.paged_attention_8bit(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["lens"], s["table"],
                                         case["D"] ** -0.5, case["most"])}


def _appended(s, q):
    """The query and the updated caches: codes of 8 bits as e4m3 numbers, beside the powers of two that they are
    multiples of."""
    out = {"q": q, "kc": s["kc"], "vc": s["vc"]}
    if s["ks"] is not None:
        out.update(ks=s["ks"], vs=s["vs"])
    return out


# ---- the operators in elementary operations ----------------------------------------------------------------------------
def _rotate(x, cos, sin, interleaved):
    """x (..., D); cos, sin broadcast to (..., R / 2); elements from R on pass."""
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., 2 * half:]), -1)


def _norm(x, w, eps=1e-6):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def _plain_norm_rotary(s):
    case, dtype = s["case"], s["q"].dtype
    at = s["positions"][:, None] if s["positions"] is not None else torch.arange(case["L"], device="cuda")
    cos, sin = s["cos"][at], s["sin"][at]
    with torch.set_grad_enabled(case["grad"]):
        x = [s[n].detach().float().requires_grad_(case["grad"]) for n in ("q", "k", "wq", "wk")]
        q = _rotate(_norm(x[0], x[2]), cos, sin, case["interleaved"])
        k = _rotate(_norm(x[1], x[3]), cos, sin, case["interleaved"])
        if not case["grad"]:
            return {"q": q.to(dtype), "k": k.to(dtype)}
        g = torch.autograd.grad((q, k), x, (s["gq"].float(), s["gk"].float()))
    return {"q": q.detach().to(dtype), "k": k.detach().to(dtype), "dq": g[0].to(dtype), "dk": g[1].to(dtype),
            "dwq": g[2].to(s["wq"].dtype), "dwk": g[3].to(s["wk"].dtype)}


def _places(s):
    """Of every row of q: its sequence, its place in it, and whether it has one."""
    rows, lens = torch.arange(s["q"].shape[0], device="cuda"), s["lens"].long()
    if s["starts"] is None:
        return rows, lens - 1, lens > 0
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, rows, right=True) - 1
    inside = seq < lens.numel()
    seq = seq.clamp(max=lens.numel() - 1)
    place = lens[seq] - (starts[seq + 1] - rows)
    return seq, place, inside & (place >= 0)


def _to_e4m3(x):
    """64-bit x, |x| <= 448, to the nearest e4m3 number, ties to even: the conversion's own rounding goes by 32 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).to(_E4M3)


def _store8(cache, scales, x, block, off):
    """Rows x (n, Hk, D) in 64 bits to places (block, off) of a cache of 8 bits."""
    blocks, Hk, BS, D = cache.shape
    amax = torch.zeros(blocks, Hk, dtype=torch.float64, device="cuda")
    amax.scatter_reduce_(0, block[:, None].expand(-1, Hk), x.abs().amax(-1), "amax")
    first = torch.full((blocks,), BS, device="cuda").scatter_reduce(0, block, off, "amin")   # its first new place
    # the least e with amax <= 448 2^e = 1.75 2^(e + 8), from amax = m 2^x with m in [0.5, 1)
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (m > 0.875).int(), _LEAST).clamp(min=_LEAST)
    need = torch.exp2(e.double())
    fresh, touched = (first == 0)[:, None], (first < BS)[:, None]
    new = torch.where(fresh, need, torch.maximum(need, scales.double()))
    grown = (touched & ~fresh & (new > scales))[:, :, None, None]
    kept = torch.arange(BS, device="cuda")[:, None] < first[:, None, None, None]
    hit = (grown & kept).expand_as(cache)
    moved = cache.double() * (scales.double() / new)[:, :, None, None]
    cache.view(torch.uint8).copy_(torch.where(hit, _to_e4m3(moved).view(torch.uint8), cache.view(torch.uint8)))
    scales.copy_(torch.where(touched, new, scales.double()))
    codes = _to_e4m3((x / new[block][..., None]).clamp(-448.0, 448.0))
    cache.view(torch.uint8)[block, :, off] = codes.view(torch.uint8)


def _plain_append(s):
    case, BS = s["case"], s["case"]["block"]
    seq, place, has = _places(s)
    at = torch.where(has, place, 0)
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q = s["q"].float()
    if s["wq"] is not None:
        q = _norm(q, s["wq"].float())
    q = torch.where(has[:, None, None], _rotate(q, cos, sin, case["interleaved"]), 0.0).to(s["q"].dtype)
    # a code of 8 bits jumps at its borders: the key is worked out in 64
    wide = torch.float64 if s["ks"] is not None else torch.float32
    k = s["k"].to(wide)
    if s["wk"] is not None:
        k = _norm(k, s["wk"].to(wide))
    k = _rotate(k, cos.to(wide), sin.to(wide), case["interleaved"])[has]
    v = s["v"][has]
    block, off = s["table"][seq[has], at[has] // BS].long(), at[has] % BS
    if s["ks"] is None:
        s["kc"][block, :, off] = k.to(s["kc"].dtype)
        s["vc"][block, :, off] = v
    else:
        _store8(s["kc"], s["ks"], k, block, off)
        _store8(s["vc"], s["vs"], v.double(), block, off)
    return _appended(s, q)


def _plain_decode(s):
    case = s["case"]
    S, H, Hk, D, BS = case["seqs"], case["H"], case["Hk"], case["D"], case["block"]
    most = max(1, max(_lengths(case)))
    table = s["table"][:, :_cdiv(most, BS)].long()
    N = table.shape[1] * BS

    def gathered(codes, scales):   # (S, Hk, N, D)
        x = codes.view(torch.uint8)[table].view(_E4M3).float() * scales[table][..., None, None]
        return x.transpose(1, 2).reshape(S, Hk, N, D)

    q = s["q"].float().view(S, Hk, H // Hk, D)
    p = torch.matmul(q, gathered(s["kc"], s["ks"]).transpose(2, 3)) * D ** -0.5
    seen = (torch.arange(N, device="cuda") < s["lens"][:, None])[:, None, None]
    p = p.masked_fill(~seen, -math.inf)
    top = p.amax(-1, keepdim=True).clamp(min=-3e38)   # (a sequence of no tokens has no maximum)
    p = torch.exp(p - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, gathered(s["vc"], s["vs"])) / torch.where(total > 0, total, 1.0)
    return {"o": o.reshape(S, H, D).to(s["q"].dtype)}


def run(s):
    if own:
        return _own(s)
    return {"norm_rotary": _plain_norm_rotary, "append": _plain_append, "decode": _plain_decode}[s["case"]["op"]](s)


# ---- the operators' definition in 64 bits ------------------------------------------------------------------------------
def _turn(x, cos, sin, interleaved, back=False):
    """The rotation (`back`: its transpose) written as products with complex numbers."""
    R = 2 * cos.shape[-1]
    z = torch.complex(cos.double(), -sin.double() if back else sin.double())
    head = x[..., :R].double()
    pairs = head.unflatten(-1, (R // 2, 2)) if interleaved else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    t = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    t = t.flatten(-2) if interleaved else t.transpose(-1, -2).flatten(-2)
    return torch.cat((t, x[..., R:].double()), -1)


def _exact_norm_rotary(s):
    case, out = s["case"], {}
    at = s["positions"][:, None] if s["positions"] is not None else torch.arange(case["L"], device="cuda")[None, None]
    cos, sin = s["cos"][at], s["sin"][at]
    for name in ("q", "k"):
        x, w = s[name].detach().double(), s["w" + name].detach().double()
        r = (x.pow(2).sum(-1, keepdim=True) / case["D"] + 1e-6) ** -0.5
        out[name] = _turn(x * r * w, cos, sin, case["interleaved"])
        if case["grad"]:
            h = _turn(s["g" + name], cos, sin, case["interleaved"], back=True)
            out["dw" + name] = (h * x * r).sum((0, 1, 2))
            a = h * w
            out["d" + name] = a * r - x * r ** 3 * (a * x).sum(-1, keepdim=True) / case["D"]
    return out


def _codes():
    """Every finite e4m3 number that is not negative, in order, and the borders between neighbours."""
    v = torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
                     dtype=torch.float64, device="cuda")
    return v, (v[1:] + v[:-1]) / 2


def _nearest(x):
    """The e4m3 number next to x; at a border the one of even index, which is the one of even mantissa."""
    v, mid = _codes()
    y = x.abs().clamp(max=448.0)
    up, down = torch.searchsorted(mid, y, right=True), torch.searchsorted(mid, y)
    return torch.copysign(v[torch.where(up % 2 == 0, up, down)], x)


def _exact_append(s):
    case, BS = s["case"], s["case"]["block"]
    past, new = _lengths(case)
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    out = {"q": q, "kc": s["kc"].double(), "vc": s["vc"].double()}
    if s["ks"] is not None:
        out.update(ks=s["ks"].double(), vs=s["vs"].double())
    table, row = s["table"].tolist(), 0
    for i, (p, n) in enumerate(zip(past, new)):
        at = torch.arange(p, p + n, device="cuda")
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        turned = []
        for name in ("q", "k"):
            x = s[name][row:row + n].double()
            if s["w" + name] is not None:
                x = x * (x.pow(2).sum(-1, keepdim=True) / case["D"] + 1e-6) ** -0.5 * s["w" + name].double()
            turned.append(_turn(x, cos, sin, case["interleaved"]))
        q[row:row + n] = turned[0]
        for name, x in (("k", turned[1]), ("v", s["v"][row:row + n].double())):
            done = 0
            while done < n:
                b, off = table[i][(p + done) // BS], (p + done) % BS
                m = min(BS - off, n - done)
                part, cache = x[done:done + m].transpose(0, 1), out[name + "c"]   # (Hk, m, D)
                done += m
                if s["ks"] is None:
                    cache[b, :, off:off + m] = part
                    continue
                scales = out[name + "s"]
                amax = part.abs().amax((1, 2)).clamp(min=448.0 * 2.0 ** _LEAST)
                e = torch.ceil(torch.log2(amax) - math.log2(448.0))
                e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)   # (the logarithm may be off by a rounding)
                e = torch.where(amax <= 448.0 * torch.exp2(e - 1), e - 1, e)
                scale = torch.exp2(e)
                if off:
                    scale = torch.maximum(scale, scales[b])
                    cache[b, :, :off] = _nearest(cache[b, :, :off] * (scales[b] / scale)[:, None, None])
                scales[b] = scale
                cache[b, :, off:off + m] = _nearest(part / scale[:, None, None])
        row += n
    return out


def _exact_decode(s):
    case = s["case"]
    Hk, D, BS = case["Hk"], case["D"], case["block"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lengths(case)):
        if not n:
            continue
        blocks = s["table"][i, :_cdiv(n, BS)].long()

        def held(codes, scales):   # (Hk, n, D)
            x = codes.view(torch.uint8)[blocks].view(_E4M3).double() * scales[blocks].double()[..., None, None]
            return x.transpose(0, 1).flatten(1, 2)[:, :n]

        q = s["q"][i].double().view(Hk, -1, D)
        p = torch.softmax(q @ held(s["kc"], s["ks"]).transpose(1, 2) * D ** -0.5, -1)
        o[i] = (p @ held(s["vc"], s["vs"])).reshape(-1, D)
    return {"o": o}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm_rotary": _exact_norm_rotary, "append": _exact_append, "decode": _exact_decode}[case["op"]](s)
