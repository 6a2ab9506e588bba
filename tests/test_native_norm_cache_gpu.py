"""The native form of qk_norm_rotary, rotary_and_cache and paged_attention_8bit against the Python form: the same bits and
layouts, which calls it takes, and what it must leave."""
import threading

import pytest
import torch

import flagattention_b200 as fa
from flagattention_b200 import _native, paged, qk_norm
from test_native_host_gpu import _same, python_form  # noqa: F401
from test_paged_8bit_gpu import made as made_decode
from test_qk_norm_gpu import made as made_norm
from test_rotary_cache_gpu import E4M3, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["bhld", "blhd", "cut"])
@pytest.mark.parametrize("wdtype", [torch.float32, torch.float16, None])
@pytest.mark.parametrize("positions", [None, "row", "batch"])
def test_norm_rotary(python_form, layout, wdtype, positions):  # noqa: F811
    q, k, gq, gk, wq, wk, cos, sin = made_norm(3, 6, 2, 70, 96, torch.float16, wdtype, 64, layout, rows=90)
    pos = None if positions is None else torch.arange(70, device="cuda", dtype=torch.int32).flip(0)
    if positions == "batch":
        pos = torch.stack([pos, pos + 3, pos + 9])
    leaves = [t.requires_grad_() for t in (q, k, wq, wk) if t is not None]
    native = _native.load().qk_norm_rotary(q, k, wq, wk, cos, sin, pos, True, 1e-5)
    assert native is not None
    assert type(native[0].grad_fn).__name__ == "CppFunction"

    def run():
        y = fa.qk_norm_rotary(q, k, wq, wk, cos, sin, pos, True, 1e-5)
        return [t.detach() for t in (*y, *torch.autograd.grad(y, leaves, (gq, gk)))]

    _same(run(), python_form(run))
    with torch.no_grad():
        y = fa.qk_norm_rotary(q, k, wq, wk, cos, sin, pos, True, 1e-5)
    assert not y[0].requires_grad and torch.equal(y[0], native[0])


def test_norm_rotary_some_gradients(python_form):  # noqa: F811
    """Only one weight, only k, no weights at all: what is asked for and nothing else."""
    for wanted in ((0,), (1,), (2,), (3,), (1, 2)):
        q, k, gq, gk, wq, wk, cos, sin = made_norm(2, 4, 2, 33, 64, torch.bfloat16, torch.float32, 64, "bhld")
        x = [q, k, wq, wk]
        for i in wanted:
            x[i].requires_grad_()

        def run():
            y = fa.qk_norm_rotary(*x, cos, sin)
            return torch.autograd.grad(y, [x[i] for i in wanted], (gq, gk))

        _same(run(), python_form(run))


@pytest.mark.parametrize("native", [True, False])
def test_norm_rotary_is_differentiable_once(native, monkeypatch):
    q, k, gq, gk, wq, wk, cos, sin = made_norm(2, 4, 2, 33, 64, torch.bfloat16, torch.float32, 64, "bhld")
    if not native:
        monkeypatch.setattr(_native, "usable", lambda x: False)
    q.requires_grad_(), wq.requires_grad_()
    y = fa.qk_norm_rotary(q, k, wq, wk, cos, sin)
    dq, dw = torch.autograd.grad(y, (q, wq), (gq, gk), create_graph=True)
    with pytest.raises(RuntimeError, match="once|twice"):
        (dq.float().sum() + dw.sum()).backward()


def test_saved_operands_are_watched():
    q, k, gq, gk, wq, wk, cos, sin = made_norm(2, 4, 2, 33, 64, torch.bfloat16, torch.float32, 64, "bhld")
    q.requires_grad_()
    y = fa.qk_norm_rotary(q, k, wq, wk, cos, sin)
    k.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, q, (gq, gk))
    y = fa.qk_norm_rotary(q, k, wq, wk, cos, sin)
    torch.autograd.grad(y, q, (gq, gk))
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(y, q, (gq, gk))


def test_gradients_reach_leaves_of_the_projection():
    """Through views of one projection, accumulated over two backward passes into .grad."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2, 50, 6 * 64, generator=gen).to(torch.bfloat16).cuda().requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    cos, sin = fa.rotary_tables(50, 64, device="cuda")

    def run():
        h = x.view(2, 50, 6, 64).transpose(1, 2)
        q, k = fa.qk_norm_rotary(h[:, :4], h[:, 4:], w, w, cos, sin)
        return (q.float().square().sum() + k.float().sum())

    run().backward()
    once = x.grad.clone(), w.grad.clone()
    run().backward()
    assert torch.equal(x.grad, 2 * once[0]) and torch.equal(w.grad, 2 * once[1])


@pytest.mark.parametrize("held", [True, False])
@pytest.mark.parametrize("starts", [True, False])
def test_rotary_and_cache(python_form, held, starts):  # noqa: F811
    b = Batch([15, 16, 33, 0], [1, 1, 1, 1] if not starts else [20, 1, 0, 5], 8, 2, 128, 16, torch.bfloat16, held, seed=1,
              starts=starts)
    d, e = b.device(), b.device()
    kc, vc = (d[n].view(E4M3) if held else d[n] for n in ("kc", "vc"))
    assert _native.load().rotary_and_cache(*b.parts(d["qkv"]), kc, vc, d["lens"], d["table"], d["cos"], d["sin"], d["starts"],
                                           None, d["wq"], d["wk"], d["ks"], d["vs"], 1e-6, False) is not None
    _same([python_form(lambda: b.call(e))], [b.call(d)])
    for n in ("kc", "vc") + (("ks", "vs") if held else ()):
        assert torch.equal(d[n], e[n])


@pytest.mark.parametrize("most", [300, 9000])
def test_paged_8bit(python_form, most):  # noqa: F811
    x = [t.cuda() for t in made_decode([300, 0, 17], 16, 2, 128, 16, torch.bfloat16)]
    call = lambda: fa.paged_attention_8bit(*x, 0.1, most)  # noqa: E731
    P = paged._plan(3, 16, 2, 16, most, 0, torch.cuda.get_device_properties(0).multi_processor_count,
                    paged._how_8bit(128))
    assert _native.load().paged_8bit(*x, 0.1, most, P[0], P[1], *(P[2] or (0, 0, 0, 0))) is not None
    _same([call()], [python_form(call)])


def test_what_is_left_to_the_python_form():
    n = _native.load()
    q, k, gq, gk, wq, wk, cos, sin = made_norm(2, 4, 2, 33, 64, torch.bfloat16, torch.float32, 64, "bhld")
    norm = lambda *a, inter=False, eps=1e-6, pos=None: n.qk_norm_rotary(*a, pos, inter, eps)  # noqa: E731
    assert norm(q, k, wq, wk, cos, sin) is not None and norm(q, k, None, None, cos, sin) is not None
    for a in ((q.float(), k.float(), wq, wk, cos, sin), (q, k.half(), wq, wk, cos, sin), (q, k, wq, None, cos, sin),
              (q, k, wq.half(), wk.half(), cos, sin), (q, k, wq, wk, cos.cpu(), sin), (q, k, wq, wk, cos.double(), sin),
              (q, k[:1], wq, wk, cos, sin), (q[0], k, wq, wk, cos, sin), (q.cpu(), k, wq, wk, cos, sin),
              (q, k, wq, wk, cos[:, ::2], sin[:, ::2]), (q[:0], k[:0], wq, wk, cos, sin)):
        assert norm(*a) is None
    assert norm(q, k, wq, wk, cos, sin, eps="x") is None and norm(q, k, wq, wk, cos, sin, inter=1) is None
    assert norm(q, k, wq, wk, cos, sin, pos=torch.zeros(32, device="cuda", dtype=torch.int64)) is None
    x = [t.cuda() for t in made_decode([300, 17], 16, 2, 128, 16, torch.bfloat16)]
    dec = lambda *a: n.paged_8bit(*a, 0.1, 512, 0, 0, 0, 0, 0, 0)  # noqa: E731
    assert dec(*x) is not None
    for i, t in ((0, x[0].float()), (0, x[0][:, :3]), (1, x[1].view(torch.uint8)), (3, x[3].half()), (4, x[4][:, :1]),
                 (5, x[5].long()), (6, x[6][:1]), (6, x[6].t().contiguous().t()), (0, x[0].cpu())):
        assert dec(*x[:i], t, *x[i + 1:]) is None, i
    # and the Python form takes what differs in form only
    ref = fa.paged_attention_8bit(*x, 0.1, 300)
    assert torch.equal(fa.paged_attention_8bit(*x[:5], x[5].long(), x[6].t().contiguous().t(), 0.1, 300), ref)
    assert torch.equal(qk_norm.qk_norm_rotary(q, k, wq, wk, cos[:, :32:1], torch.cat((sin, sin), 1)[:, :32])[0],
                       fa.qk_norm_rotary(q, k, wq, wk, cos, sin)[0])


def test_several_threads_and_streams():
    """Two threads on streams of their own, forward and backward and decoding, many times: everybody's own workspace."""
    x = [t.cuda() for t in made_decode([1900, 0, 170], 16, 2, 128, 16, torch.bfloat16)]
    q, k, gq, gk, wq, wk, cos, sin = made_norm(2, 8, 2, 700, 128, torch.bfloat16, torch.float32, 128, "bhld")

    def work():
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        y = fa.qk_norm_rotary(*leaves, cos, sin)
        return [*y, *torch.autograd.grad(y, leaves, (gq, gk)), fa.paged_attention_8bit(*x, 0.1, 9000)]

    want, wrong = work(), []
    torch.cuda.synchronize()

    def run():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = work()
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(1)

    threads = [threading.Thread(target=run) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
