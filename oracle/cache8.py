"""TEST INFRASTRUCTURE ONLY: norm and rotation of heads, the paged cache's fused writer and decoding over a cache of 8 bits,
in 64 bits on the CPU, row by row.  The reference has none of them; each function states the operator's definition.
"""
import math

import torch

E4M3_MAX = 448.0


def _rotate(x, cos, sin, interleaved, back=False):
    """x (..., D) in 64 bits, cos and sin (..., R / 2); `back`: by the opposite angles."""
    half = cos.shape[-1]
    c, s = cos.double(), -sin.double() if back else sin.double()
    y = x.clone()
    lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    return y


def _angle_rows(table, positions, B, L):
    if positions is None:
        positions = torch.arange(L)
    positions = positions.cpu().long().reshape(-1, L).expand(B, L).clamp(0, table.shape[0] - 1)
    return table.cpu()[positions][:, None]


def norm_rotary(x, weight, cos, sin, positions=None, interleaved=False, eps=1e-6):
    """x (B, heads, L, D) -> 64 bits."""
    x = x.detach().cpu().double()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r if weight is None else x * r * weight.detach().cpu().double()
    B, _, L, _ = x.shape
    return _rotate(n, _angle_rows(cos, positions, B, L), _angle_rows(sin, positions, B, L), interleaved)


def norm_rotary_backward(x, weight, g, cos, sin, positions=None, interleaved=False, eps=1e-6):
    """(dx, dweight, sizes of the terms of dx, of dweight) in 64 bits: the sizes are what rounding errors go by."""
    x, g = x.detach().cpu().double(), g.cpu().double()
    B, _, L, D = x.shape
    w = torch.ones(D, dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    c, s = _angle_rows(cos, positions, B, L), _angle_rows(sin, positions, B, L)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    h = _rotate(g, c, s, interleaved, back=True)
    h_size = _rotate(g.abs(), c.abs(), -s.abs(), interleaved, back=True).abs().maximum(
        _rotate(g.abs(), c.abs(), s.abs(), interleaved, back=True).abs())
    dx = r * (h * w - x * r * r * (h * w * x).mean(-1, keepdim=True))
    size = r * (h_size * w.abs() + x.abs() * r * r * (h_size * w.abs() * x.abs()).mean(-1, keepdim=True))
    return dx, (h * x * r).sum((0, 1, 2)), size, (h_size * x.abs() * r).sum((0, 1, 2))


def to_e4m3(x):
    """The nearest e4m3 number of every 64-bit x, ties to the even mantissa; beyond +-448 that."""
    x = x.double()
    y = x.abs().clamp(max=E4M3_MAX)
    _, e = torch.frexp(torch.where(y > 0, y, 1.0))
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    y = torch.round(y / step) * step       # torch.round: ties to even
    return torch.where(torch.isnan(x), x, torch.copysign(y.clamp(max=E4M3_MAX), x))


def scale_for(values):
    """The least power of two, from 2^-126 on, that holds the finite ones of `values` as e4m3 numbers."""
    finite = values[torch.isfinite(values)].abs()
    most = float(finite.max()) if finite.numel() else 0.0
    e = -126
    while most > E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rotary_and_cache(query, key, value, key_cache, value_cache, context_lens, block_tables, cos, sin, query_starts=None,
                     positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, key_scales=None,
                     value_scales=None):
    """On CPU tensors: caches and scales in 64 bits (codes as numbers), changed in place; returns the queries in 64 bits."""
    T, Hk, BS = key.shape[0], key.shape[1], key_cache.shape[2]
    out = torch.zeros(query.shape, dtype=torch.float64)
    lens = context_lens.tolist()
    starts = list(range(T + 1)) if query_starts is None else query_starts.tolist()
    for s, length in enumerate(lens):
        rows = [r for r in range(starts[s], min(starts[s + 1], T))]
        placed = {}
        for r in rows:
            place = length - (starts[s + 1] - r)
            if place < 0 or place // BS >= block_tables.shape[1]:
                continue
            pos = place if positions is None else int(positions[r])
            pos = min(max(pos, 0), cos.shape[0] - 1)
            turned = []
            for x, w in ((query[r], q_weight), (key[r], k_weight)):
                x = x.double()
                if w is not None:
                    x = x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)) * w.double()
                turned.append(_rotate(x, cos[pos], sin[pos], interleaved))
            out[r] = turned[0]
            placed.setdefault(place // BS, []).append((place % BS, turned[1], value[r].double()))
        for logical, tokens in placed.items():
            b = int(block_tables[s, logical])
            if b < 0 or b >= key_cache.shape[0]:
                continue
            first = tokens[0][0]
            for which, (cache, scales) in ((1, (key_cache, key_scales)), (2, (value_cache, value_scales))):
                for h in range(Hk):
                    new = torch.stack([t[which][h] for t in tokens])
                    if scales is None:
                        cache[b, h, first:first + len(tokens)] = new
                        continue
                    scale, old = scale_for(new), float(scales[b, h])
                    if first and old > scale:
                        scale = old
                    if first and scale > old:
                        cache[b, h, :first] = to_e4m3(cache[b, h, :first] * (old / scale))
                    scales[b, h] = scale
                    cache[b, h, first:first + len(tokens)] = to_e4m3(new / scale)
    return out


def paged_attention_8bit(query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables, scale):
    """On CPU tensors, codes and scales of any float type: (output, sum of |weight * value|, largest sum of |q * k| * scale
    of a head, by query head) in 64 bits; the last two are what rounding errors go by."""
    S, H, D = query.shape
    Hk, BS = key_cache.shape[1:3]
    out, size = torch.zeros(S, H, D, dtype=torch.float64), torch.zeros(S, H, D, dtype=torch.float64)
    most = torch.zeros(S, H, 1, dtype=torch.float64)
    for s, n in enumerate(context_lens.tolist()):
        if n <= 0:
            continue
        ids = block_tables[s, :math.ceil(n / BS)].long()
        k = (key_cache[ids].double() * key_scales[ids].double()[..., None, None]).transpose(0, 1).reshape(Hk, -1, D)[:, :n]
        v = (value_cache[ids].double() * value_scales[ids].double()[..., None, None]).transpose(0, 1)
        v = v.reshape(Hk, -1, D)[:, :n]
        q = query[s].double().view(Hk, -1, D)
        p = torch.softmax(q @ k.transpose(1, 2) * scale, -1)
        out[s] = (p @ v).reshape(H, D)
        size[s] = (p @ v.abs()).reshape(H, D)
        most[s] = (q.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1).reshape(H, 1)
    return out, size, most
