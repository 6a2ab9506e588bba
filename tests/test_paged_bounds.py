"""Bounds of the context length up to the largest that the calls take: a caller without a bound of its own gives such a one."""
import ctypes
import random

import pytest
import torch

from flagattention_b200 import _C, paged


def test_partitions_of_8_bit_calls_under_any_bound():
    """What the library asks of sizes (paged_parts.cuh: sizing_ok) and of the grid, for bounds up to 2^31 - 1."""
    rng = random.Random(2)
    for i in range(4000):
        Hk = rng.choice([1, 2, 4, 5, 8])
        seqs, G, D = rng.choice([1, 2, 3, 8, 37, 64, 300, 3000]), rng.choice([1, 4, 8, 16, 17, 40]), rng.choice([16, 64, 128, 256])
        most = 2 ** 31 - 1 if i % 10 == 0 else int(2 ** rng.uniform(16, 31))
        size, P, sizing = paged._plan(seqs, G * Hk, Hk, 16, most, 0, 148, paged._how_8bit(D))
        finest, coarsest, ctas, parts = sizing
        assert P <= 65535 and size <= 1 << 24 and coarsest <= 1 << 24
        assert P * size >= most > (P - 1) * size and size % 16 == finest % 16 == 0 and 0 < finest <= size
        for x in (size, coarsest):
            assert x % finest == 0 and (x // finest) & (x // finest - 1) == 0 and x >= finest
        assert ctas >= 0 and (ctas > 0 or parts > 0) and (ctas == 0 or seqs <= 2048)


@pytest.mark.parametrize("most,size", [(2 ** 31 - 1, 1 << 24), (2 ** 31 - 1, 1 << 30), (2 ** 31 - 100, 4096), (1, 16), (4097, 4096)])
def test_the_workspace_of_large_bounds(built_lib, most, size):
    lib = _C.load()
    a = _C.PagedArgs()
    a.num_seqs, a.num_q_heads, a.head_size, a.max_context_len, a.partition_size = 3, 8, 64, most, size
    lib.fa_paged_workspace_bytes.restype = ctypes.c_int64
    rows = 3 * 8 * -(-most // size)
    assert lib.fa_paged_workspace_bytes(ctypes.byref(a)) == rows * 64 * 4 + 2 * rows * 4


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [0, 1, 2, 300])
@pytest.mark.parametrize("seqs", [2, 40])
def test_8_bit_decoding_without_a_bound(seqs, splits):
    from test_paged_8bit_gpu import call, check, made
    gen = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 2000, (seqs,), generator=gen).tolist()
    x = made(lens, 8, 2, 64, 16, torch.bfloat16, seed=seqs)
    check(call(x, 0.125, 2 ** 31 - 1, splits), x, 0.125)
    with pytest.raises(AssertionError):
        call(x, 0.125, 2 ** 31, splits)
