"""What qk_norm_rotary, rotary_and_cache and paged_attention_8bit refuse, before anything is launched; no GPU needed.

Checks of tensors that need a GPU are at the end, marked for one; the library's own are called through the C ABI."""
import ctypes

import pytest
import torch

import flagattention_b200 as fa
from flagattention_b200 import _C

E4M3 = torch.float8_e4m3fn


def test_norm_rotary_refuses():
    x = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    cos, sin = fa.rotary_tables(8, 64)
    w = torch.ones(64)
    q, k = x(1, 4, 8, 64), x(1, 2, 8, 64)
    for bad in ((q[0], k), (q, x(2, 2, 8, 64)), (q, x(1, 2, 7, 64)), (q, x(1, 2, 8, 32)), (x(1, 4, 8, 40), x(1, 2, 8, 40)),
                (x(1, 4, 8, 528), x(1, 2, 8, 528)), (x(1, 0, 8, 64), k), (q, x(1, 0, 8, 64))):
        with pytest.raises(AssertionError):
            fa.qk_norm_rotary(*bad, w, w, cos, sin)
    with pytest.raises(AssertionError, match="CUDA"):
        fa.qk_norm_rotary(q, k, w, w, cos, sin)


def test_tables_and_weights_are_checked():
    from flagattention_b200 import qk_norm
    cpu = torch.device("cpu")
    cos, sin = fa.rotary_tables(8, 64)
    qk_norm.check_tables(cos, sin, 64, cpu)
    qk_norm.check_tables(cos[:, :16], sin[:, :16], 64, cpu)
    for bad in ((cos.double(), sin), (cos, sin[:7]), (cos[0], sin[0]), (cos[:, :4], sin[:, :4]), (cos[:, :0], sin[:, :0]),
                (cos[:0], sin[:0])):
        with pytest.raises(AssertionError):
            qk_norm.check_tables(*bad, 64, cpu)
    with pytest.raises(AssertionError):
        qk_norm.check_tables(cos, sin, 48, cpu)                  # more than the head has
    with pytest.raises(AssertionError):
        qk_norm.check_tables(cos, sin, 64, torch.device("cuda", 0))
    like = torch.zeros(1, dtype=torch.bfloat16)
    w = torch.ones(64)
    assert qk_norm.check_weights(None, None, 64, like) == (None, None)
    got = qk_norm.check_weights(torch.ones(65)[1:], w, 64, like)
    assert all(t.data_ptr() % 16 == 0 for t in got)              # moved to where the kernels can read it
    for bad in ((w, None), (None, w), (w, w.bfloat16()), (w.half(), w.half()), (w.double(), w.double()), (w[:32], w)):
        with pytest.raises(AssertionError):
            qk_norm.check_weights(*bad, 64, like)


def _decode(**change):
    a = dict(query=torch.zeros(2, 8, 64, dtype=torch.float16), key_cache=torch.zeros(6, 2, 16, 64, dtype=E4M3),
             value_cache=torch.zeros(6, 2, 16, 64, dtype=E4M3), key_scales=torch.ones(6, 2), value_scales=torch.ones(6, 2),
             context_lens=torch.ones(2, dtype=torch.int32), block_tables=torch.zeros(2, 3, dtype=torch.int32),
             attn_scale=0.1, max_context_len=48)
    a.update(change)
    return a


def test_host_tensors_are_refused():
    with pytest.raises(AssertionError, match="CUDA"):
        fa.paged_attention_8bit(**_decode())
    a = _decode()
    with pytest.raises(AssertionError, match="CUDA"):
        fa.rotary_and_cache(a["query"], a["query"][:, :2], a["query"][:, :2], a["key_cache"], a["value_cache"],
                            a["context_lens"], a["block_tables"], *fa.rotary_tables(8, 64), key_scales=a["key_scales"],
                            value_scales=a["value_scales"])


def _norm_args(**change):
    a = _C.NormRotaryArgs(_C.FA_BF16, 1, 4, 2, 8, 64, 64, 0, 1, 8, 1e-6, 0x1000, 0x1000, 0x1000, 0x1000, None, 0)
    for n, v in change.items():
        setattr(a, n, v)
    return ctypes.byref(a)


def test_library_checks_norm_rotary(built_lib):
    lib = _C.load()
    lib.fa_qk_norm_rotary_bwd_workspace_bytes.restype = ctypes.c_int64
    t, off = _C.Tensor4(0x1000, 0, 0, 64), _C.Tensor4(0x1008, 0, 0, 64)
    odd = _C.Tensor4(0x1000, 0, 0, 63)
    r = ctypes.byref

    def fwd(a, q=t):
        return lib.fa_qk_norm_rotary_fwd(a, r(q), r(t), r(t), r(t), None)

    assert lib.fa_qk_norm_rotary_fwd(None, r(t), r(t), r(t), r(t), None) == -1
    for change, status in ((dict(dtype=7), -1), (dict(H=0), -1), (dict(Hk=-1), -1), (dict(B=-1), -1), (dict(table_rows=0), -1),
                           (dict(cos=None), -1), (dict(D=72), -2), (dict(D=528), -2), (dict(rotary_dim=72), -2),
                           (dict(rotary_dim=80), -2), (dict(cos=0x1004), -3), (dict(q_weight=0x1008), -3)):
        assert fwd(_norm_args(**change)) == status, change
    assert fwd(_norm_args(), off) == -3 and fwd(_norm_args(), odd) == -3
    assert fwd(_norm_args(B=0)) == 0 and fwd(_norm_args(L=0)) == 0
    p = ctypes.c_void_p
    size = lib.fa_qk_norm_rotary_bwd_workspace_bytes(_norm_args())
    assert size > 0 and size % (64 * 4) == 0 and lib.fa_qk_norm_rotary_bwd_workspace_bytes(_norm_args(D=72)) == 0

    def bwd(ws, n, g=t):
        return lib.fa_qk_norm_rotary_bwd(_norm_args(), r(t), r(t), r(g), r(t), r(t), r(t), p(0x1000), None, ws,
                                         ctypes.c_int64(n), None)

    assert bwd(None, size) == -5 and bwd(p(0x1000), size - 1) == -5 and bwd(p(0x1004), size) == -5
    assert bwd(p(0x1000), size, off) == -3


def _cache_args(**change):
    a = _C.RotaryCacheArgs()
    base = dict(dtype=_C.FA_F16, num_tokens=3, num_seqs=3, num_q_heads=4, num_kv_heads=2, head_size=64, rotary_dim=64,
                block_size=16, num_blocks=4, table_cols=2, table_rows=8, eps=1e-6, query=0x1000, key=0x1000, value=0x1000,
                out=0x1000, key_cache=0x1000, value_cache=0x1000, context_lens=0x1000, block_tables=0x1000, cos=0x1000,
                sin=0x1000)
    base.update(change)
    for n, v in base.items():
        setattr(a, n, v)
    return ctypes.byref(a)


def test_library_checks_rotary_cache(built_lib):
    lib = _C.load()
    assert lib.fa_rotary_cache(None, None) == -1
    for change, status in ((dict(dtype=2), -1), (dict(num_tokens=-1), -1), (dict(num_seqs=2), -1), (dict(block_size=0), -1),
                           (dict(head_size=48, rotary_dim=48), -2), (dict(head_size=512), -2), (dict(rotary_dim=80), -2),
                           (dict(rotary_dim=24), -2), (dict(query=None), -1), (dict(block_tables=None), -1),
                           (dict(key_scales=0x1000), -1), (dict(k_weight=0x1000), -1), (dict(key=0x1008), -3),
                           (dict(v_stride_t=12), -3), (dict(kv_stride_b=8 * 3 + 4), -3),
                           (dict(key_scales=0x1000, value_scales=0x1000, kv_stride_t=8), -3)):
        assert lib.fa_rotary_cache(_cache_args(**change), None) == status, change
    assert lib.fa_rotary_cache(_cache_args(num_tokens=0, num_seqs=0), None) == 0


def test_library_checks_paged_8bit(built_lib):
    lib = _C.load()

    def call(sizing=(0, 0, 0, 0), key_scales=0x1000, num_blocks=4, table_cols=2, **change):
        a = _C.Paged8bitArgs()
        base = dict(dtype=_C.FA_F16, num_seqs=3, num_q_heads=4, num_kv_heads=2, head_size=64, block_size=16,
                    max_context_len=512, query=0x1000, key_cache=0x1000, value_cache=0x1000, context_lens=0x1000,
                    block_tables=0x1000, out=0x1000, kv_stride_t=64)
        base.update(change)
        for n, v in base.items():
            setattr(a.paged, n, v)
        a.key_scales, a.value_scales, a.num_blocks, a.table_cols = key_scales, 0x1000, num_blocks, table_cols
        return lib.fa_paged_attention_8bit(ctypes.byref(a), *sizing, None)

    parts = dict(partition_size=256, part_out=0x1000, part_max=0x1000, part_sum=0x1000)
    assert lib.fa_paged_attention_8bit(None, 0, 0, 0, 0, None) == -1
    for change, status in ((dict(dtype=5), -1), (dict(num_seqs=0), -1), (dict(num_q_heads=5), -1), (dict(block_size=24), -1),
                           (dict(partition_size=24), -1), (dict(causal_rows=1), -1), (dict(block_table_is_i64=2), -1),
                           (dict(head_size=48), -2), (dict(head_size=512), -2), (dict(key_cache=0x1008), -3),
                           (dict(kv_stride_t=8), -3), (dict(q_stride_h=12), -3), (dict(partition_size=256), -5),
                           (dict(context_lens=None), -1), (dict(key_scales=None), -1), (dict(num_blocks=-1), -1),
                           (dict(num_q_heads=200000, num_kv_heads=100000), -6), (dict(table_cols=0), -1),
                           (dict(num_seqs=1 << 27, num_q_heads=64, num_kv_heads=32), -6)):
        assert call(**change) == status, change
    for sizing in ((24, 256, 0, 1), (256, 128, 0, 1), (96, 256, 0, 1), (256, 512, -1, 1), (256, 512, 0, 0)):
        assert call(sizing, **parts) == -1, sizing
    assert call((256, 512, 100, 0), num_blocks=4, **dict(parts, num_seqs=3000)) == -1


def test_packed_structs():
    """The byte strings that the operators pass, against the ctypes declarations, field by field in order."""
    for packer, struct in ((_C.NORM_ROTARY_ARGS, _C.NormRotaryArgs), (_C.ROTARY_CACHE_ARGS, _C.RotaryCacheArgs)):
        kinds = [k for _, k in struct._fields_]
        values = [0.5 if k is ctypes.c_float else i + 1 for i, k in enumerate(kinds)]
        got = struct.from_buffer_copy(packer.pack(*values))
        assert [getattr(got, n) for n, _ in struct._fields_] == values
    values = list(range(1, 10)) + [0.5] + list(range(10, 28))
    got = _C.Paged8bitArgs.from_buffer_copy(_C.PAGED_8BIT_ARGS.pack(*values, 100, 101, 102, 103))
    assert [getattr(got.paged, n) for n, _ in _C.PagedArgs._fields_] == values
    assert (got.key_scales, got.value_scales, got.num_blocks, got.table_cols) == (100, 101, 102, 103)


def test_partitions_of_8_bit_calls_are_what_the_library_takes():
    """Sizes nest, cover the bound and are whole groups of tokens, for any call (paged_parts.cuh: sizing_ok)."""
    import random
    from flagattention_b200 import paged
    rng = random.Random(1)
    for _ in range(3000):
        Hk = rng.choice([1, 2, 4, 5, 8])
        seqs, G, D = rng.choice([1, 2, 3, 8, 37, 64, 300, 3000]), rng.choice([1, 4, 8, 16, 17, 40]), rng.choice([16, 64, 128, 256])
        block, most = rng.choice([16, 32, 48, 128, 512]), int(2 ** rng.uniform(0, 20))
        size, P, sizing = paged._plan(seqs, G * Hk, Hk, block, most, 0, 148, paged._how_8bit(D))
        if not size:
            assert sizing is None
            continue
        finest, coarsest, ctas, parts = sizing
        assert P * size >= most > (P - 1) * size and size % 16 == finest % 16 == 0 and 0 < finest <= size
        for x in (size, coarsest):
            assert x % finest == 0 and (x // finest) & (x // finest - 1) == 0 and x >= finest
        assert ctas >= 0 and (ctas > 0 or parts > 0) and (ctas == 0 or seqs <= 2048)
    # one long context: one wave of CTAs
    size, P, sizing = paged._plan(1, 64, 8, 32, 131072, 0, 148, paged._how_8bit(128))
    assert 8 * P <= 3 * 148 < 8 * P * 2 and sizing[3] == 55


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    """The checks behind `is_cuda`, with nothing launched."""
    def gpu(a):
        return {n: v.cuda() if torch.is_tensor(v) else v for n, v in a.items()}

    out = fa.paged_attention_8bit(**gpu(_decode(context_lens=torch.zeros(2, dtype=torch.int32))))
    assert (out == 0).all()
    z = torch.zeros
    for change in (dict(query=z(2, 8, 48, dtype=torch.float16)), dict(query=z(2, 7, 64, dtype=torch.float16)),
                   dict(query=z(2, 8, 64)), dict(key_cache=z(6, 2, 16, 64, dtype=torch.float16)),
                   dict(value_cache=z(5, 2, 16, 64, dtype=E4M3)), dict(key_scales=torch.ones(6, 1)),
                   dict(value_scales=torch.ones(6, 2).double()), dict(value_scales=torch.ones(2, 6).t()),
                   dict(context_lens=torch.ones(3, dtype=torch.int32)), dict(context_lens=torch.ones(2)),
                   dict(block_tables=z(3, 3, dtype=torch.int32)), dict(block_tables=z(2, 3, dtype=torch.int16)),
                   dict(max_context_len=0), dict(num_splits=-1),
                   dict(key_cache=z(6, 2, 24, 64, dtype=E4M3), value_cache=z(6, 2, 24, 64, dtype=E4M3))):
        with pytest.raises(AssertionError):
            fa.paged_attention_8bit(**gpu(_decode(**change)))
    with pytest.raises(AssertionError):
        fa.paged_attention_8bit(**{**gpu(_decode()), "block_tables": _decode()["block_tables"]})

    def write(**change):
        a = dict(query=z(2, 8, 64, dtype=torch.float16), key=z(2, 2, 64, dtype=torch.float16),
                 value=z(2, 2, 64, dtype=torch.float16), key_cache=z(6, 2, 16, 64, dtype=E4M3),
                 value_cache=z(6, 2, 16, 64, dtype=E4M3), context_lens=torch.ones(2, dtype=torch.int32),
                 block_tables=z(2, 3, dtype=torch.int32), cos=torch.ones(4, 32), sin=torch.ones(4, 32),
                 key_scales=torch.ones(6, 2), value_scales=torch.ones(6, 2))
        a.update(change)
        return fa.rotary_and_cache(**gpu(a))

    write()
    for change in (dict(key=z(2, 3, 64, dtype=torch.float16)), dict(value=z(2, 2, 32, dtype=torch.float16)),
                   dict(key=z(2, 2, 64, dtype=torch.bfloat16)), dict(key_scales=None), dict(value_scales=None),
                   dict(key_cache=z(6, 2, 16, 64, dtype=torch.float16), value_cache=z(6, 2, 16, 64, dtype=torch.float16)),
                   dict(context_lens=torch.ones(1, dtype=torch.int32), block_tables=z(1, 3, dtype=torch.int32)),
                   dict(query_starts=torch.ones(2, dtype=torch.int32)), dict(query_starts=torch.ones(3)),
                   dict(positions=torch.ones(2)), dict(positions=torch.ones(3, dtype=torch.int64)),
                   dict(cos=torch.ones(4, 48), sin=torch.ones(4, 48)), dict(q_weight=torch.ones(64)),
                   dict(block_tables=z(1, 3, dtype=torch.int32)), dict(key_scales=torch.ones(6, 3))):
        with pytest.raises(AssertionError):
            write(**change)


@pytest.mark.gpu
def test_calls_without_heads_blocks_or_angles_are_refused():
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    h, c = z(2, 4, 64, dtype=torch.float16), z(6, 4, 16, 64, dtype=torch.float16)
    lens, bt, ang = z(2, dtype=torch.int32), z(2, 3, dtype=torch.int32), torch.ones(4, 32, device="cuda")
    fa.rotary_and_cache(h, h, h, c, c.clone(), lens, bt, ang, ang)
    for args in ((h[:, :0], h, h, c, c, lens, bt, ang, ang), (h, h[:, :0], h[:, :0], c[:, :0], c[:, :0], lens, bt, ang, ang),
                 (h, h, h, c[:0], c[:0], lens, bt, ang, ang), (h, h, h, c[:, :, :0], c[:, :, :0], lens, bt, ang, ang),
                 (h, h, h, c, c, lens, bt, ang[:0], ang[:0]), (h, h, h, c, c, lens, bt, ang[:, :0], ang[:, :0])):
        with pytest.raises(AssertionError):
            fa.rotary_and_cache(*args)
    q = z(2, 4, 3, 64, dtype=torch.float16)
    for args in ((q[:, :0], q, None, None, ang, ang), (q, q[:, :0], None, None, ang, ang),
                 (q, q, None, None, ang[:0], ang[:0]), (q, q, None, None, ang[:, :0], ang[:, :0]),
                 (q[..., :0], q[..., :0], None, None, ang[:, :0], ang[:, :0])):
        with pytest.raises(AssertionError):
            fa.qk_norm_rotary(*args)
    e = z(6, 2, 16, 64, dtype=E4M3)
    s = z(6, 2)
    for args in ((h[:, :0], e, e, s, s), (h, e[:, :0], e[:, :0], s[:, :0], s[:, :0]), (h, e[:0], e[:0], s[:0], s[:0]),
                 (h, e[:, :, :0], e[:, :, :0], s, s)):
        with pytest.raises(AssertionError):
            fa.paged_attention_8bit(*args, lens, bt, 0.1, 48)
