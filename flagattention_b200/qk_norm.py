"""qk_norm_rotary: RMS norm of every head of queries and keys and their rotation by position, in one pass.

The step between a decoder's projections and flash_attention.  No reference counterpart: its operators take queries and
keys as they are.  One HBM-bound launch forward for q and k together; one backward, and a small one that adds up the
weights' gradients, in an order that depends on the shape and the GPU's number of SMs: the same bits every time.
"""
import torch

from . import _C, _native, rotary

__all__ = ["qk_norm_rotary"]


def check_tables(cos, sin, head_dim, device):
    """cos, sin for the kernels and the rows they have: fp32 (positions, half of the rotated elements)."""
    for t in (cos, sin):
        assert t.device == device, \
            f"cos / sin tables are on {t.device}, the operands on {device} (rotary_tables(..., device=q.device))"
        assert t.dtype == torch.float32 and t.dim() == 2, "cos / sin tables are fp32 (positions, rotated elements / 2)"
    assert cos.shape == sin.shape and cos.shape[0] > 0, "cos / sin tables must share their shape"
    assert 0 < 2 * cos.shape[1] <= head_dim and cos.shape[1] % 8 == 0, \
        "the rotated elements are a multiple of 16, at most head_dim"
    return aligned(cos), aligned(sin)


def check_weights(q_weight, k_weight, head_dim, like):
    """Both weights for the kernels, (None, None) for none."""
    assert (q_weight is None) == (k_weight is None), "weights for q and k, or for neither"
    if q_weight is None:
        return None, None
    for w in (q_weight, k_weight):
        assert w.shape == (head_dim,), "a weight has head_dim elements"
        assert w.dtype in (torch.float32, like.dtype) and w.dtype == q_weight.dtype, \
            "weights are both fp32 or both of the operands' type"
        assert w.device == like.device, f"weights are on {w.device}, the operands on {like.device}"
    return aligned(q_weight), aligned(k_weight)


def aligned(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _like(x):
    y = torch.empty_like(x)
    return y if _C.kernel_ready(y) is y else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _pack(q, k, q_weight, k_weight, cos, sin, positions, pos_stride, interleaved, eps):
    B, H, L, D = q.shape
    return _C.NORM_ROTARY_ARGS.pack(
        _C.dtype_code(q.dtype), B, H, k.shape[1], L, D, 2 * cos.shape[1], 1 if interleaved else 0,
        1 if q_weight is not None and q_weight.dtype == torch.float32 else 0, cos.shape[0], eps, _ptr(q_weight),
        _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), _ptr(positions), pos_stride)


class QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps):
        assert q.dim() == 4 and k.dim() == 4, "q and k are (batch, heads, length, head_dim)"
        B, H, L, D = q.shape
        assert k.shape[0] == B and k.shape[2:] == q.shape[2:], "q and k share batch, length and head_dim"
        assert H > 0 and k.shape[1] > 0, "q and k have heads"
        assert D > 0 and D % 16 == 0 and D <= 512, "head_dim must be a multiple of 16, at most 512"
        assert q.is_cuda, "q must be a CUDA tensor"
        assert k.device == q.device and k.dtype == q.dtype, "q and k share device and type"
        dtype = _C.dtype_code(q.dtype)  # noqa: F841  (asserts the type)
        cos, sin = check_tables(cos, sin, D, q.device)
        w = check_weights(q_weight, k_weight, D, q)
        pos, _, pos_stride = rotary._positions_ready(positions, B, L, q.device)
        q, k = _C.kernel_ready(q), _C.kernel_ready(k)
        q_out, k_out = _like(q), _like(k)
        with _C.device_guard(q.device):
            st = _C.call("fa_qk_norm_rotary_fwd")(
                _pack(q, k, *w, cos, sin, pos, pos_stride, interleaved, eps), _C.pack4(q), _C.pack4(k),
                _C.pack4(q_out), _C.pack4(k_out), _C.raw_stream(q.device))
        _C.check(st, "fa_qk_norm_rotary_fwd")
        ctx.save_for_backward(q, k, *w, cos, sin, pos)
        ctx.args = (pos_stride, bool(interleaved), float(eps))
        return q_out, k_out

    @staticmethod
    def backward(ctx, gq, gk):
        with torch.no_grad():
            grads = QkNormRotary._gradients(ctx, gq, gk)
        if torch.is_grad_enabled():   # an error for whoever goes through these gradients again, with or without gq's graph
            given = [g.detach().requires_grad_() for g in grads if g is not None]
            marked = iter(torch._C._functions.DelayedError(b"qk_norm_rotary is differentiable once", len(given))(*given))
            grads = [None if g is None else next(marked) for g in grads]
        return (*grads, None, None, None, None, None)

    @staticmethod
    def _gradients(ctx, gq, gk):
        q, k, wq, wk, cos, sin, pos = ctx.saved_tensors
        pos_stride, interleaved, eps = ctx.args
        gq, gk = _C.kernel_ready(gq), _C.kernel_ready(gk)
        dq, dk = _like(q), _like(k)
        dwq = torch.empty_like(wq) if wq is not None and ctx.needs_input_grad[2] else None
        dwk = torch.empty_like(wk) if wk is not None and ctx.needs_input_grad[3] else None
        with _C.device_guard(q.device):
            args = _pack(q, k, wq, wk, cos, sin, pos, pos_stride, interleaved, eps)
            size, ws = 0, None
            if dwq is not None or dwk is not None:
                size = _C.call("fa_qk_norm_rotary_bwd_workspace_bytes")(args)
                ws = torch.empty(size, dtype=torch.uint8, device=q.device)
            st = _C.call("fa_qk_norm_rotary_bwd")(
                args, _C.pack4(q), _C.pack4(k), _C.pack4(gq), _C.pack4(gk), _C.pack4(dq), _C.pack4(dk), _ptr(dwq),
                _ptr(dwk), _ptr(ws), size, _C.raw_stream(q.device))
        _C.check(st, "fa_qk_norm_rotary_bwd")
        return [dq, dk, dwq, dwk]


def qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions=None, interleaved=False, eps=1e-6):
    """Returns (q', k'): every head of q and k RMS-normed and rotated, the operands of flash_attention.

    q: (batch, heads, length, head_dim), k: (batch, kv_heads, length, head_dim), fp16 / bf16, head_dim a multiple of 16 up
    to 512.  x' = rotate(x * rsqrt(mean(x^2) + eps) * weight).  q_weight, k_weight: (head_dim,) of that type or fp32, or
    both None for ones.  cos, sin: fp32 (num_positions, rotated / 2): the first `rotated` elements of a head turn (a
    multiple of 16, at most head_dim), in pairs (i, i + rotated / 2) or, interleaved, (2i, 2i + 1); the others only are
    normed.  positions: None (token l sits at position l) or integers of shape (length,) or (batch, length); values outside
    the tables are clamped.  fp32 arithmetic, results rounded once.  Differentiable (once) with respect to q, k and the
    weights; the weights' gradients are the same bits every time."""
    if _native.usable(q):
        pair = _native.load().qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps)
        if pair is not None:
            return pair
    return QkNormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps)
