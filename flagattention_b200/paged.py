"""paged_attention: single-token decode over a block-table KV cache.

Mirrors src/flag_attn/paged.py:6-163: same arguments, same split rule
(num_splits == 0 picks it automatically, 1 disables it, > 1 fixes the count),
returns a new tensor shaped like `query`.
"""
import ctypes
import functools
import math

import torch

from . import _C, _native
from .qk_norm import check_tables, check_weights

__all__ = ["attention", "attention_8bit", "reshape_and_cache", "rotary_and_cache"]


def _next_power_of_2(n):
    return 1 << (max(int(n), 1) - 1).bit_length()


def _cdiv(a, b):
    return (a + b - 1) // b


def plan_partitions(num_seqs, num_kv_heads, kv_block_size, max_context_len, num_splits, num_sms):
    """Returns (num_splits, partition_size) by the reference's rule
    (src/flag_attn/paged.py:40-53); partition_size is 0 when there is one pass."""
    partition_size = 0
    if num_splits == 0:
        if num_seqs * num_kv_heads > 2 * num_sms:
            num_splits = 1
            if max_context_len >= 4096:
                partition_size = max(256, kv_block_size)
                num_splits = _cdiv(max_context_len, partition_size)
        else:
            partition_size = max(256, kv_block_size)
            num_splits = _cdiv(max_context_len, partition_size)
            if max_context_len <= 1024 or kv_block_size >= 256:
                num_splits = 1
    elif num_splits > 1:
        partition_size = _next_power_of_2(_cdiv(max_context_len, num_splits))
    if num_splits == 1:
        partition_size = 0
    return num_splits, partition_size


def coarsen_partition(partition_size, pairs, context_len, num_sms, most=2048):
    """Partitions of `partition_size` tokens, doubled up to `most` while `pairs` contexts of `context_len` tokens, one
    CTA a partition, keep the GPU busy with them.

    A CTA's four warps fill a ring of loads and merge their results once per partition, and every partition writes and
    re-reads a row of fp32 partial output, so short ones cost bandwidth; fewer CTAs than SMs cost more (fp16, one
    context of 32768 over 4 kv heads: 256: 54 us, 512: 37, 1024: 33, 2048: 40)."""
    while partition_size < most and pairs * _cdiv(int(context_len), 2 * partition_size) >= 0.8 * num_sms:
        partition_size *= 2
    return partition_size


@functools.lru_cache(maxsize=1024)
def size_partitions(base, num_seqs, ctas, max_context_len, num_sms, fill=0.8, many=35, top=2048, slots=0):
    """(workspace partition, finest, coarsest, ctas, parts) of a fa_paged_attention call: how far partitions of `base`
    tokens may grow when max_context_len is an upper bound and lengths differ.  `ctas`: CTAs that a partition of one
    sequence takes; workspace partition 0: one pass does it.

    The workspace partition is the largest at which one sequence still has CTAs enough for the GPU, or until the grid is
    down to 35 CTAs an SM: doubling lengthens the longest partition (1 us per 100 tokens of a CTA by itself) and spares
    half the launches (1 ns each).  Shorter sequences are cut finer on the GPU: into two waves' worth each where there
    are fewer sequences than that; or, where the workspace partition had to stay small but many sequences might fill
    larger ones, by the sum of all lengths (both kernels then read every length: below 1 us).  fp16, head_size 128, us;
    256 tokens each / sized by the bound as if every context had it / this:
      8 kv heads   4 x 1500 under 32768 15 / 20 / 10, 16 x 2048 at most 22 / 27 / 20, 4096 and 63 x 200 35 / 36 / 31,
                   64 x 32768 at most 852 / 642 / 647, 64 x 8192 at most 233 / 189 / 192, 4 x 32768 at most 103 / 74 / 75
      2 kv heads   4 x 1500 under 32768 9.5 / 21 / 10.3, 4096 and 63 x 200 16.5 / 26 / 17.5, 16 x 32768 at most
                   96 / 52 / 55, 32768 and 15 x 1000 44 / 33 / 32, 64 x 32768 at most 253 / 159 / 174"""
    pairs = num_seqs * ctas
    if slots and max_context_len < 4096 and (pairs > 2 * num_sms or max_context_len <= 1024):
        # short contexts: four waves of CTAs at most, and partitions that are long where one pass fills the GPU already
        # (codes of 8 bits, one pass -> this, us: 8 kv heads, 16 x 3000 tokens 33 -> 27, 40 x 1-3000 42 -> 32, 64 x 1-3000
        # 50 -> 46, 100 x 3000 112 -> 104; 1 kv head, 16 x 1-1000 19 -> 11.4; contexts far below the bound pay 3 us)
        size = base if 2 * pairs <= slots * num_sms else 2 * base if pairs <= slots * num_sms else 8 * base
        while size < max_context_len and pairs * _cdiv(max_context_len, size) > 4 * slots * num_sms:
            size *= 2
        return (0, base, base, 0, 1) if max_context_len <= size else (size, size, size, 0, _cdiv(max_context_len, size))
    if 16 * pairs <= slots * num_sms < pairs * _cdiv(max_context_len, base):
        # few long contexts: one wave of equal partitions, `slots` CTAs an SM (131071 tokens, 8 kv heads, codes of 8 bits, an
        # earlier kernel: 59 us so, 76 with the power of two below, 71 with the one above)
        parts = slots * num_sms // pairs
        finest = size = min(max(base, _cdiv(_cdiv(max_context_len, parts), 128) * 128), 1 << 24)   # (what the library takes)
        while finest % 32 == 0 and finest >= 256:   # for contexts far below the bound
            finest //= 2
        return (0, base, base, 0, 1) if max_context_len <= size else (size, finest, size, 0, parts)
    coarsest = base
    while coarsest < top:
        coarsest *= 2
    size = base
    while size < coarsest and (ctas * _cdiv(max_context_len, 2 * size) >= fill * num_sms
                               or num_seqs * ctas * _cdiv(max_context_len, size) > many * num_sms):
        size *= 2
    while slots and _cdiv(max_context_len, size) > 4096:   # bounds that are none: of the workspace, and of the grid (65535)
        size *= 2
    coarsest = max(coarsest, size)
    if max_context_len <= size:
        return 0, base, coarsest, 0, 1
    pairs = num_seqs * ctas
    by_length = (size < min(coarsest, 4 * base) and num_seqs <= 2048
                 and pairs * _cdiv(max_context_len, 2 * size) >= fill * num_sms)
    if by_length:
        return size, base, coarsest, int(fill * num_sms), 0
    return size, base if pairs < 2 * num_sms else size, coarsest, 0, max(1, _cdiv(2 * num_sms, pairs))


def partition_workspace(rows, P, D, device):
    """One allocation for the partial results of `rows` (sequence, query head) rows over P partitions:
    (tensor, address of the outputs (rows, P, D), of the maxima (rows, P), of the sums (rows, P)), all fp32."""
    stats = (rows * P + 63) // 64 * 64
    ws = torch.empty(rows * P * D + 2 * stats, dtype=torch.float32, device=device)
    base = ws.data_ptr()
    part_max = base + rows * P * D * 4
    return ws, base, part_max, part_max + stats * 4


def _plan(num_seqs, num_q_heads, num_kv_heads, kv_block_size, max_context_len, num_splits, num_sms, how=()):
    """(partition size, partitions of the workspace, sizing or None) of a call; partition size 0: one pass."""
    # kept for plain numbers only: a tensor hashes by identity, and its value may change
    plan = _kept_plan if type(num_splits) is int else _kept_plan.__wrapped__
    return plan(num_seqs, num_q_heads, num_kv_heads, kv_block_size, max_context_len, num_splits, num_sms, how)


@functools.lru_cache(maxsize=1024)
def _kept_plan(num_seqs, num_q_heads, num_kv_heads, kv_block_size, max_context_len, num_splits, num_sms, how=()):
    free_choice = num_splits == 0
    num_splits, partition_size = plan_partitions(num_seqs, num_kv_heads, kv_block_size, max_context_len, num_splits,
                                                 num_sms)
    sizing = None
    if free_choice and (partition_size or how):
        partition_size, *sizing = size_partitions(
            256 if how else partition_size, num_seqs, num_kv_heads * _cdiv(num_q_heads // num_kv_heads, 16),
            max_context_len, num_sms, *how)
    if not partition_size:
        return 0, 0, None
    return partition_size, _cdiv(max_context_len, partition_size), sizing


def attention(query, key_cache, value_cache, context_lens, block_tables, attn_scale,
              max_context_len, num_splits=0):
    """query [num_seqs, kv_heads * group, head]; caches [num_blocks, kv_heads, block, head]
    with identical strides; context_lens [num_seqs] int32; block_tables
    [num_seqs, max_blocks] int32 or int64."""
    if type(max_context_len) is int and max_context_len > 0 and num_splits == 0 and _native.usable(query):
        out = _native_attention(query, key_cache, value_cache, context_lens, block_tables, attn_scale, max_context_len)
        if out is not None:
            return out
    num_seqs, num_q_heads, head_size = query.shape
    num_kv_heads, kv_block_size = key_cache.shape[1], key_cache.shape[2]
    assert key_cache.shape[3] == head_size
    assert num_q_heads % num_kv_heads == 0
    query_group_size = num_q_heads // num_kv_heads
    assert head_size in (16, 32, 64, 128, 256, 512), f"head_size={head_size}"
    assert head_size <= 256, "head_size 512 is not built for B200 yet"
    assert query_group_size == 1 or kv_block_size >= 16, f"kv_block_size={kv_block_size}"
    assert key_cache.stride() == value_cache.stride(), "key and value cache must share strides"
    assert query.is_cuda and query.dtype == key_cache.dtype == value_cache.dtype
    assert block_tables.dtype in (torch.int32, torch.int64)
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache),
                    ("context_lens", context_lens), ("block_tables", block_tables)):
        assert t.device == query.device, f"{name} is on {t.device}, query on {query.device}"

    if context_lens.dtype != torch.int32:
        context_lens = context_lens.to(torch.int32)
    context_lens = context_lens.contiguous()
    if block_tables.stride(-1) != 1:
        block_tables = block_tables.contiguous()
    if query.stride(-1) != 1 or query.data_ptr() % 16 or query.stride(0) % 8 or query.stride(1) % 8:
        query = query.contiguous()
    if key_cache.stride(-1) != 1 or any(s % 8 for s in key_cache.stride()[:-1]):
        key_cache, value_cache = key_cache.contiguous(), value_cache.contiguous()

    with _C.device_guard(query.device):
        partition_size, P, sizing = _plan(num_seqs, num_q_heads, num_kv_heads, kv_block_size, int(max_context_len),
                                          num_splits, _C.sm_count(query.device))
        part_out = part_max = part_sum = 0
        if partition_size:
            assert partition_size >= kv_block_size and partition_size % kv_block_size == 0, \
                f"partition_size={partition_size}, kv_block_size={kv_block_size}"
            assert partition_size % 16 == 0, f"partition_size={partition_size}"
            ws, part_out, part_max, part_sum = partition_workspace(
                num_seqs * num_q_heads, P, head_size, query.device)

        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        kb, kh, kt = key_cache.stride()[:3]
        args = _C.PAGED_ARGS.pack(
            _C.dtype_code(query.dtype), num_seqs, num_q_heads, num_kv_heads, head_size, kv_block_size,
            int(max_context_len), 1 if block_tables.dtype == torch.int64 else 0, partition_size, attn_scale,
            query.data_ptr(), query.stride(0), query.stride(1), key_cache.data_ptr(), value_cache.data_ptr(), kb, kh, kt,
            context_lens.data_ptr(), block_tables.data_ptr(), block_tables.stride(0),
            out.data_ptr(), out.stride(0), out.stride(1), part_out, part_max, part_sum, 0)
        stream = _C.raw_stream(query.device)
        if sizing and partition_size:
            _C.check(_C.call("fa_paged_attention")(args, *sizing, stream), "fa_paged_attention")
            return out
        _C.check(_C.call("fa_paged_decode")(args, stream), "fa_paged_decode")
        if partition_size:
            _C.check(_C.call("fa_paged_reduce")(args, stream), "fa_paged_reduce")
    return out


def _native_attention(query, key_cache, value_cache, context_lens, block_tables, attn_scale, max_context_len):
    """The call through native code, or None: partitions and their workspace chosen here, the rest there."""
    if query.dim() != 3 or key_cache.dim() != 4:
        return None
    num_seqs, num_q_heads, head_size = query.shape
    num_kv_heads, kv_block_size = key_cache.shape[1:3]
    if not num_seqs or not num_kv_heads or num_q_heads % num_kv_heads or not kv_block_size or head_size > 256:
        return None
    partition_size, P, sizing = _plan(num_seqs, num_q_heads, num_kv_heads, kv_block_size, max_context_len, 0,
                                      _C.sm_count(query.device))
    part_out = part_max = part_sum = 0
    if partition_size:
        ws, part_out, part_max, part_sum = partition_workspace(num_seqs * num_q_heads, P, head_size, query.device)
    return _native.load().paged(query, key_cache, value_cache, context_lens, block_tables, attn_scale, max_context_len,
                                partition_size, part_out, part_max, part_sum, *(sizing or (0, 0, 0, 0)))


def reshape_and_cache(key, value, key_cache, value_cache, slot_mapping):
    """Writes new tokens into the paged caches `attention` reads.

    key, value: [num_tokens, kv_heads, head]; caches [num_blocks, kv_heads, block, head];
    slot_mapping [num_tokens] integer: token i goes to block slot // block, position slot % block;
    negative slots are skipped.  The reference has no writer (its tests fill the caches with random
    numbers); a serving loop runs this step right before the decode kernel."""
    if _native.usable(key) and _native.load().append(key, value, key_cache, value_cache, slot_mapping):
        return
    num_tokens, num_kv_heads, head_size = key.shape
    assert value.shape == key.shape and key_cache.shape == value_cache.shape
    assert key_cache.shape[1] == num_kv_heads and key_cache.shape[3] == head_size
    assert key.dtype == value.dtype == key_cache.dtype == value_cache.dtype
    assert key_cache.stride() == value_cache.stride(), "key and value cache must share strides"
    assert key_cache.stride(-1) == 1 and all(s % 8 == 0 for s in key_cache.stride()[:-1]), \
        "caches need unit inner stride and 16-byte aligned rows"
    assert slot_mapping.numel() == num_tokens
    assert key.is_cuda, "inputs must be CUDA tensors"
    for name, t in (("value", value), ("key_cache", key_cache), ("value_cache", value_cache),
                    ("slot_mapping", slot_mapping)):
        assert t.device == key.device, f"{name} is on {t.device}, key on {key.device}"
    if key.stride() != value.stride() or key.stride(-1) != 1 or any(s % 8 for s in key.stride()[:-1]) \
            or key.data_ptr() % 16 or value.data_ptr() % 16:
        key, value = key.contiguous(), value.contiguous()
    slots = slot_mapping.to(torch.int64).contiguous()
    kb, kh, kt = key_cache.stride()[:3]
    with _C.device_guard(key.device):
        st = _C.call("fa_paged_cache_append")(
            _C.dtype_code(key.dtype), num_tokens, num_kv_heads, head_size, key_cache.shape[2], key.data_ptr(),
            value.data_ptr(), key.stride(0), key.stride(1), key_cache.data_ptr(), value_cache.data_ptr(), kb, kh, kt,
            slots.data_ptr(), _C.raw_stream(key.device))
    _C.check(st, "fa_paged_cache_append")


# ---- caches of 8 bits --------------------------------------------------------------------------------------------------
def _check_scales(key_cache, key_scales, value_scales):
    for t in (key_scales, value_scales):
        assert t.dtype == torch.float32 and t.shape == key_cache.shape[:2] and t.is_contiguous(), \
            "scales are contiguous fp32 [num_blocks, kv_heads]"
        assert t.device == key_cache.device, f"scales are on {t.device}, the caches on {key_cache.device}"


def _check_caches(key_cache, value_cache, num_kv_heads, head_size, unit):
    """What both writers and readers of caches with a table ask: `unit` elements are 16 bytes."""
    assert key_cache.dim() == 4 and key_cache.shape == value_cache.shape
    assert key_cache.shape[0] > 0, "caches have blocks"
    assert key_cache.shape[1] == num_kv_heads and key_cache.shape[3] == head_size
    assert key_cache.dtype == value_cache.dtype
    assert key_cache.device == value_cache.device, "the caches are on one device"
    assert key_cache.stride() == value_cache.stride(), "key and value cache must share strides"
    assert key_cache.stride(-1) == 1 and all(s % unit == 0 for s in key_cache.stride()[:-1]) \
        and key_cache.data_ptr() % 16 == 0 and value_cache.data_ptr() % 16 == 0, \
        "caches need unit inner stride and 16-byte aligned rows"


def _table_ready(block_tables, num_seqs, device):
    assert block_tables.dtype in (torch.int32, torch.int64) and block_tables.dim() == 2
    assert block_tables.shape[0] == num_seqs and block_tables.device == device
    return block_tables if block_tables.stride(1) == 1 or block_tables.shape[1] <= 1 else block_tables.contiguous()


def _int32(t, name, n, device):
    assert t.device == device, f"{name} is on {t.device}, the operands on {device}"
    assert not t.is_floating_point() and t.shape == (n,), f"{name} has {n} integers"
    return t.to(torch.int32).contiguous()


def _rows_ready(t):
    """Unit inner stride, 16-byte aligned rows."""
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0 and all(
        s % 8 == 0 or n <= 1 for n, s in zip(t.shape[:2], t.stride()[:2]))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _two_parts(x):
    """A number as fp32 and what that leaves out, fp32 as well."""
    high = ctypes.c_float(x).value
    return high, float(x) - high if math.isfinite(high) else 0.0


def _stride(t, i):
    return t.stride(i) if t.shape[i] > 1 else 0


def _how_8bit(head_size):
    """(fill, many, top, slots) of size_partitions for caches of 8 bits.

    A token's bytes are half and a CTA's work on it is not, so partitions end where more CTAs an SM are at hand, and
    may be longer; the size of a block does not matter.  16-bit rule -> this, us (an earlier kernel): 37 x 1-8191 tokens,
    2 kv heads of 16, head 64 34 -> 25, 64 x 1K-32K, 8 kv heads of 4, head 128 439 -> 422, 2 x 8000 19.6 -> 15, 1 x 30000
    in blocks of 256 334 -> 22.  One wave of 3 CTAs an SM where 4 fit: one of 131071 51, of 4 56."""
    return 3, 35, 4096, 4 if head_size <= 64 else 3 if head_size <= 128 else 2


def attention_8bit(query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables, attn_scale,
                   max_context_len, num_splits=0):
    """`attention` over caches held in 8 bits: key_cache, value_cache [num_blocks, kv_heads, block, head] of
    torch.float8_e4m3fn, key_scales, value_scales [num_blocks, kv_heads] fp32, 0 or positive; a value is code * scale.

    query [num_seqs, kv_heads * group, head] fp16 / bf16, head 16, 32, 64, 128 or 256; block a multiple of 16;
    context_lens [num_seqs] and block_tables [num_seqs, max_blocks] as in `attention`.  A sequence of length 0 gives 0;
    one whose table names a block that the cache does not have gives NaN.  fp32 sums and statistics, the output rounded
    once.  `rotary_and_cache` writes such caches.  Not differentiable: operands that require gradients give an output that
    does not.  Several rows of one sequence (a chunk of a prompt) are given as sequences of their own, each with its place + 1
    as its length and its sequence's row of the table; each reads the cache once."""
    if type(max_context_len) is int and max_context_len > 0 and num_splits == 0 and _native.usable(query):
        out = _native_8bit(query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables, attn_scale,
                           max_context_len)
        if out is not None:
            return out
    assert query.dim() == 3
    num_seqs, num_q_heads, head_size = query.shape
    assert query.is_cuda, "query must be a CUDA tensor"
    dtype = _C.dtype_code(query.dtype)
    num_kv_heads, kv_block_size = key_cache.shape[1], key_cache.shape[2]
    assert num_kv_heads > 0 and num_q_heads > 0 and num_q_heads % num_kv_heads == 0
    assert head_size in (16, 32, 64, 128, 256), f"head_size={head_size}"
    assert key_cache.dtype == torch.float8_e4m3fn, "caches of torch.float8_e4m3fn"
    assert kv_block_size > 0 and kv_block_size % 16 == 0, f"kv_block_size={kv_block_size}"
    assert key_cache.device == query.device, f"key_cache is on {key_cache.device}, query on {query.device}"
    _check_caches(key_cache, value_cache, num_kv_heads, head_size, 16)
    _check_scales(key_cache, key_scales, value_scales)
    max_context_len = int(max_context_len)
    assert 0 < max_context_len < 2 ** 31 and num_splits >= 0
    context_lens = _int32(context_lens, "context_lens", num_seqs, query.device)
    block_tables = _table_ready(block_tables, num_seqs, query.device)
    query = _rows_ready(query)
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if num_seqs == 0 or block_tables.shape[1] == 0:
        return out.zero_()
    with _C.device_guard(query.device):
        partition_size, P, sizing = _plan(num_seqs, num_q_heads, num_kv_heads, kv_block_size, max_context_len, num_splits,
                                          _C.sm_count(query.device), _how_8bit(head_size))
        part_out = part_max = part_sum = 0
        if partition_size:
            assert partition_size % 16 == 0, f"partition_size={partition_size}"
            ws, part_out, part_max, part_sum = partition_workspace(num_seqs * num_q_heads, P, head_size, query.device)
        kb, kh, kt = key_cache.stride()[:3]
        args = _C.PAGED_8BIT_ARGS.pack(
            dtype, num_seqs, num_q_heads, num_kv_heads, head_size, kv_block_size, max_context_len,
            1 if block_tables.dtype == torch.int64 else 0, partition_size, attn_scale, query.data_ptr(),
            _stride(query, 0), _stride(query, 1), key_cache.data_ptr(), value_cache.data_ptr(), kb, kh, kt,
            context_lens.data_ptr(), block_tables.data_ptr(), block_tables.stride(0), out.data_ptr(), out.stride(0),
            out.stride(1), part_out, part_max, part_sum, 0, key_scales.data_ptr(), value_scales.data_ptr(),
            key_cache.shape[0], block_tables.shape[1])
        st = _C.call("fa_paged_attention_8bit")(args, *(sizing or (0, 0, 0, 0)), _C.raw_stream(query.device))
    _C.check(st, "fa_paged_attention_8bit")
    return out


def _native_8bit(query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables, attn_scale,
                 max_context_len):
    """The call through native code, or None; the partitions are chosen here."""
    if query.dim() != 3 or key_cache.dim() != 4:
        return None
    num_seqs, num_q_heads, head_size = query.shape
    num_kv_heads, kv_block_size = key_cache.shape[1:3]
    if not num_seqs or not num_q_heads or not num_kv_heads or num_q_heads % num_kv_heads or not kv_block_size:
        return None
    partition_size, P, sizing = _plan(num_seqs, num_q_heads, num_kv_heads, kv_block_size, max_context_len, 0,
                                      _C.sm_count(query.device), _how_8bit(head_size))
    return _native.load().paged_8bit(query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables,
                                     attn_scale, max_context_len, partition_size, P, *(sizing or (0, 0, 0, 0)))


def rotary_and_cache(query, key, value, key_cache, value_cache, context_lens, block_tables, cos, sin, query_starts=None,
                     positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, key_scales=None,
                     value_scales=None):
    """Writes the new tokens of a batch of sequences into the paged caches, keys rotated (and normed) on the way, and
    returns their queries rotated (and normed): the step in front of `attention` or `attention_8bit`.

    query [num_tokens, heads, head], key, value [num_tokens, kv_heads, head], fp16 / bf16, head 16, 32, 64, 128 or 256.
    context_lens [num_seqs] counts the new tokens, as the attention that follows takes it; sequence s has rows
    query_starts[s] .. query_starts[s + 1] - 1 (integers [num_seqs + 1], ascending), the last of them its last token (those from
    num_tokens on are not there); None: one row a sequence.  block_tables [num_seqs, max_blocks].  A row's position in the tables is its place in its sequence,
    or positions [num_tokens], clamped to them.  cos, sin, weights, eps, interleaved: as in qk_norm_rotary, no norm
    without weights.

    Caches [num_blocks, kv_heads, block, head] of the operands' type, or of torch.float8_e4m3fn with key_scales,
    value_scales [num_blocks, kv_heads] fp32: a block's scale starts with its first token, is the least power of two
    that holds its values, and earlier codes are brought along when it grows, so that a block filled token by token is one
    filled at once (but for codes below 2^-6, which lose bits on the way).  Infinities are held as +-448 times the scale.

    Rows behind the last sequence, or in front of theirs (context_lens smaller than its rows; 0 for an idle slot of a
    padded batch), are written nowhere and come back as 0.  A block that is written to must belong to one sequence only:
    otherwise what its places hold afterwards is not defined.  Not differentiable: operands that require gradients give an
    output that does not."""
    if _native.usable(query):
        out = _native.load().rotary_and_cache(query, key, value, key_cache, value_cache, context_lens, block_tables, cos,
                                              sin, query_starts, positions, q_weight, k_weight, key_scales, value_scales,
                                              eps, interleaved)
        if out is not None:
            return out
    assert query.dim() == key.dim() == value.dim() == 3
    num_tokens, num_q_heads, head_size = query.shape
    num_kv_heads = key.shape[1]
    assert value.shape == key.shape and key.shape[0] == num_tokens and key.shape[2] == head_size
    assert query.is_cuda, "query must be a CUDA tensor"
    dtype = _C.dtype_code(query.dtype)
    assert query.dtype == key.dtype == value.dtype
    assert num_q_heads > 0 and num_kv_heads > 0
    assert head_size in (16, 32, 64, 128, 256), f"head_size={head_size}"
    device = query.device
    for name, t in (("key", key), ("value", value), ("key_cache", key_cache)):
        assert t.device == device, f"{name} is on {t.device}, query on {device}"
    held = key_cache.dtype == torch.float8_e4m3fn
    assert held or key_cache.dtype == query.dtype, "caches of the operands' type or of torch.float8_e4m3fn"
    assert (key_scales is not None) == (value_scales is not None) == held, "scales belong to caches of 8 bits"
    _check_caches(key_cache, value_cache, num_kv_heads, head_size, 16 if held else 8)
    assert key_cache.shape[2] > 0
    if held:
        _check_scales(key_cache, key_scales, value_scales)
    num_seqs = context_lens.shape[0]
    context_lens = _int32(context_lens, "context_lens", num_seqs, device)
    block_tables = _table_ready(block_tables, num_seqs, device)
    assert query_starts is not None or num_tokens == num_seqs, "one row a sequence, or query_starts"
    if query_starts is not None:
        query_starts = _int32(query_starts, "query_starts", num_seqs + 1, device)
    if positions is not None:
        assert not positions.is_floating_point() and positions.shape == (num_tokens,), "positions are num_tokens integers"
        assert positions.device == device, f"positions are on {positions.device}, query on {device}"
        positions = positions.to(torch.int64).contiguous()
    cos, sin = check_tables(cos, sin, head_size, device)
    q_weight, k_weight = check_weights(q_weight, k_weight, head_size, query)
    query, key, value = _rows_ready(query), _rows_ready(key), _rows_ready(value)
    out = torch.empty(query.shape, dtype=query.dtype, device=device)
    if num_tokens == 0:
        return out
    if num_seqs == 0 or block_tables.shape[1] == 0:   # no row has a place
        return out.zero_()

    def ptr(t):
        return 0 if t is None else t.data_ptr()

    kb, kh, kt = key_cache.stride()[:3]
    args = _C.ROTARY_CACHE_ARGS.pack(
        dtype, num_tokens, num_seqs, num_q_heads, num_kv_heads, head_size, 2 * cos.shape[1], 1 if interleaved else 0,
        key_cache.shape[2], key_cache.shape[0], block_tables.shape[1], 1 if block_tables.dtype == torch.int64 else 0,
        cos.shape[0], 1 if q_weight is not None and q_weight.dtype == torch.float32 else 0, *_two_parts(eps),
        *(x for t in (query, key, value, out) for x in (t.data_ptr(), _stride(t, 0), _stride(t, 1))),
        key_cache.data_ptr(), value_cache.data_ptr(), kb, kh, kt, ptr(key_scales), ptr(value_scales),
        context_lens.data_ptr(), ptr(query_starts), block_tables.data_ptr(), block_tables.stride(0), ptr(positions),
        cos.data_ptr(), sin.data_ptr(), ptr(q_weight), ptr(k_weight))
    with _C.device_guard(device):
        st = _C.call("fa_rotary_cache")(args, _C.raw_stream(device))
    _C.check(st, "fa_rotary_cache")
    return out
