"""What attention's queries and keys go through before they are attended, on MI355X: a
root-mean-square norm of each head and the rotation by position, in one pass over both.

    y = x (mean x^2 + eps)^(-1/2) (weight_offset + weight)         over a head's D values
    (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)           over pairs of the first R

The pairs are (i, R / 2 + i), or (2 i, 2 i + 1) with interleaved=True; the R are twice the
columns of the tables cos and sin, whose row i holds the angles of position i (rope_tables
makes them). Everything is float32 inside and rounded once. Forward, and backward through
autograd, in float32, bfloat16 and float16; on the GPU only, a missing library or a CPU
tensor raises.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import _dtype_code, _launch, _no_tangents, _one_device, _plan, _steps, _untraced
from .gated_deltanet import _aligned, grad_needed

MAX_WIDTH = 256  # of a head


def rope_tables(positions: int, rotary: int, base: float = 10000.0, device="cuda"):
    """cos and sin [positions, rotary / 2] float32 of the angles position / base^(2 i / rotary),
    taken in float64: angles of far positions lose nothing but the tables' own rounding."""
    if rotary % 2 or rotary < 0 or positions < 0:
        raise ValueError("rotary must be even, neither it nor positions negative")
    i = torch.arange(0, rotary, 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / max(rotary, 1))
    return angle.cos().float(), angle.sin().float()


def _rope_sizes(q, k, dtype, k_dtype, qw, kw, w_dtype, kw_dtype, cos, sin, cos_dtype, sin_dtype, positions, pos_dtype):
    """Checked sizes (B, T, Hq, Hk, D, R) of a call with tensors of these shapes and types."""
    if len(q) != 4 or len(k) != 4 or q[:2] != k[:2] or q[3] != k[3]:
        raise ValueError("expected q [B,T,Hq,D] and k [B,T,Hk,D]")
    batch, length, hq, d = q
    hk = k[2]
    if hq < 1 or hk < 1 or d < 1:
        raise ValueError("q and k need at least one head of at least one value")
    if d > MAX_WIDTH:
        raise ValueError(f"no kernel for head widths above {MAX_WIDTH} (got {d})")
    if qw != (d,) or kw != (d,):
        raise ValueError("expected a weight [D] for q and for k")
    if k_dtype != dtype or kw_dtype != w_dtype:
        raise ValueError("q and k must have one dtype, and their weights one")
    _dtype_code(dtype), _dtype_code(w_dtype)
    if len(cos) != 2 or sin != cos or cos_dtype != torch.float32 or sin_dtype != torch.float32:
        raise ValueError("expected float32 tables cos and sin [positions, R / 2] of one shape")
    if 2 * cos[1] > d:
        raise ValueError("the tables rotate more values than a head has")
    if pos_dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    if len(positions) not in (1, 2) or positions[-1] not in (1, length) or (
            len(positions) == 2 and positions[0] not in (1, batch)):
        raise ValueError("expected positions [T] or [B,T] (or what broadcasts to it)")
    return batch, length, hq, hk, d, 2 * cos[1]


@_plan
def _rope_plan(q_stride, k_stride, pos_stride, *call):
    """_rope_sizes of a call, the dtype codes of its rows and weights, the stride arrays of
    the rows (None if an innermost axis is not dense) and of the positions, and whether those
    have 64 bits."""
    sizes = _rope_sizes(*call)
    q, k, positions = call[0], call[1], call[12]
    if max(*q, *k, call[8][0]) >= 2**31:
        raise ValueError("q, k and the tables must have less than 2^31 rows an axis")
    dense = all(x[3] == 1 or stride[3] == 1 for x, stride in ((q, q_stride), (k, k_stride)))
    lead = 2 - len(positions)
    pos_steps = _steps(((1,) * lead + tuple(positions) + (1,), (0,) * lead + tuple(pos_stride) + (1,)))
    return (sizes, _dtype_code(call[2]), _dtype_code(call[6]), _steps((q, q_stride), (k, k_stride)) if dense else None,
            pos_steps, int(call[13] == torch.int64))


def _call(q, k, q_weight, k_weight, cos, sin, positions):
    return (q.shape, k.shape, q.dtype, k.dtype, q_weight.shape, k_weight.shape, q_weight.dtype, k_weight.dtype, cos.shape,
            sin.shape, cos.dtype, sin.dtype, positions.shape, positions.dtype)


def _operands(q, k, q_weight, k_weight, cos, sin, positions, weight_offset, *grads):
    """The device, the checked sizes, the tensors as the kernels read them (to be kept until
    the launch) and the arguments that name them."""
    args = (q, k, q_weight, k_weight, cos, sin, positions)
    plan = _rope_plan(q.stride(), k.stride(), positions.stride(), *_call(*args))
    dev = _one_device(*args, *grads)
    if (plan[3] is None or (q.data_ptr() | k.data_ptr() | q_weight.data_ptr() | k_weight.data_ptr() | cos.data_ptr()
                            | sin.data_ptr()) % 16
            or not (q_weight.is_contiguous() and k_weight.is_contiguous() and cos.is_contiguous() and sin.is_contiguous())):
        # (the strides are taken last: a copy for the alignment may have others than its view)
        q, k = (_aligned(x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous(), 16) for x in (q, k))
        args = (q, k, *(_aligned(x.contiguous(), 16) for x in args[2:6]), positions)
        plan = _rope_plan(q.stride(), k.stride(), positions.stride(), *_call(*args))
    sizes, code, wcode, steps, pos_steps, pos64 = plan
    return dev, sizes, args, (q.data_ptr(), k.data_ptr(), code, steps, args[2].data_ptr(), args[3].data_ptr(), wcode,
                              weight_offset, args[4].data_ptr(), args[5].data_ptr(), cos.shape[0], positions.data_ptr(),
                              pos64, pos_steps)


def _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, weight_offset, interleaved):
    dev, sizes, kept, args = _operands(q, k, q_weight, k_weight, cos, sin, positions, weight_offset)
    q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
    _launch("pbattn_qk_norm_rope", _lib.attn_lib().pbattn_qk_norm_rope, dev, *args, q_out.data_ptr(), k_out.data_ptr(), *sizes,
            eps, int(interleaved))
    return q_out, k_out


@_plan
def _workspace_size(width: int, device_index: int) -> int:
    with torch.cuda.device(device_index):  # (the size depends on the device's compute units)
        return _lib.attn_lib().pbattn_qk_norm_rope_bwd_workspace_size(width)


def _gradient(x, grad):
    """The gradient of a result as the kernel reads it: dense, in x's dtype."""
    if grad.shape != x.shape:
        raise ValueError("grad_q and grad_k must have q's and k's shapes")
    if grad.dtype == x.dtype and grad.is_contiguous() and not grad.data_ptr() % 16:
        return grad
    return _aligned(grad.to(x.dtype).contiguous(), 16)


def _backward(q, k, q_weight, k_weight, cos, sin, positions, grad_q, grad_k, eps, weight_offset, interleaved):
    dev, sizes, kept, args = _operands(q, k, q_weight, k_weight, cos, sin, positions, weight_offset, grad_q, grad_k)
    grad_q, grad_k = _gradient(q, grad_q), _gradient(k, grad_k)
    dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
    dqw, dkw = q_weight.new_empty(sizes[4]), k_weight.new_empty(sizes[4])
    if sizes[0] == 0 or sizes[1] == 0:
        return dq, dk, dqw.zero_(), dkw.zero_()
    nbytes = _workspace_size(sizes[4], dev.index)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch("pbattn_qk_norm_rope_bwd", _lib.attn_lib().pbattn_qk_norm_rope_bwd, dev, *args, grad_q.data_ptr(),
            grad_k.data_ptr(), dq.data_ptr(), dk.data_ptr(), dqw.data_ptr(), dkw.data_ptr(), *sizes, eps, int(interleaved),
            workspace.data_ptr(), nbytes)
    return dq, dk, dqw, dkw


@torch.library.custom_op("pbgdn::qk_norm_rope", mutates_args=(),
                         schema="(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos, Tensor sin, "
                                "Tensor positions, float eps, float weight_offset, bool interleaved) -> (Tensor, Tensor)")
def qk_norm_rope_op(q, k, q_weight, k_weight, cos, sin, positions, eps, weight_offset, interleaved):
    """qk_norm_rope, for graphs of ops."""
    return _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, weight_offset, interleaved)


@qk_norm_rope_op.register_fake
def _(q, k, q_weight, k_weight, cos, sin, positions, eps, weight_offset, interleaved):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("pbgdn::qk_norm_rope_backward", mutates_args=(),
                         schema="(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos, Tensor sin, "
                                "Tensor positions, Tensor grad_q, Tensor grad_k, float eps, float weight_offset, "
                                "bool interleaved) -> (Tensor, Tensor, Tensor, Tensor)")
def qk_norm_rope_backward_op(q, k, q_weight, k_weight, cos, sin, positions, grad_q, grad_k, eps, weight_offset, interleaved):
    """(dq, dk, dq_weight, dk_weight) of qk_norm_rope."""
    return _backward(q, k, q_weight, k_weight, cos, sin, positions, grad_q, grad_k, eps, weight_offset, interleaved)


@qk_norm_rope_backward_op.register_fake
def _(q, k, q_weight, k_weight, cos, sin, positions, grad_q, grad_k, eps, weight_offset, interleaved):
    return tuple(x.new_empty(x.shape) for x in (q, k, q_weight, k_weight))


def _setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:7])
    ctx.rest = inputs[7:]
    ctx.set_materialize_grads(False)


def _gradients(backward):
    """The backward formula, by `backward`: the op, or its launch itself."""
    def formula(ctx, grad_q, grad_k):
        if grad_q is None and grad_k is None:
            return (None,) * 10
        saved = ctx.saved_tensors
        grad_q = torch.zeros_like(saved[0]) if grad_q is None else grad_q
        grad_k = torch.zeros_like(saved[1]) if grad_k is None else grad_k
        return *backward(*saved, grad_q, grad_k, *ctx.rest), None, None, None, None, None, None
    return formula


qk_norm_rope_op.register_autograd(_gradients(qk_norm_rope_backward_op), setup_context=_setup)


class _QkNormRope(torch.autograd.Function):
    """The op and its gradients without the op's dispatch, which costs more than a short call."""
    _launched = staticmethod(_gradients(_backward))
    _traced = staticmethod(_gradients(qk_norm_rope_backward_op))

    @staticmethod
    def forward(ctx, *inputs):
        output = _forward(*inputs)
        _setup(ctx, inputs, output)
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        _no_tangents("qk_norm_rope's backward", grad_q, grad_k)
        tensors = [t for t in (grad_q, grad_k) if t is not None]
        return (_QkNormRope._launched if _untraced(*tensors) else _QkNormRope._traced)(ctx, grad_q, grad_k)


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps: float = 1e-6, *, weight_offset: float = 0.0,
                 interleaved: bool = False):
    """Queries q [B,T,Hq,D] and keys k [B,T,Hk,D] (one dtype, any strides; D up to 256) normed
    over each head with q_weight and k_weight [D] (weight_offset added to both: 1.0 for
    weights kept about zero) and their first R values rotated: cos, sin [P, R / 2] float32
    by positions (int32 or int64, [T] or [B,T] or what broadcasts to it). A token whose
    position is not in the tables (-1: padding) gets zeros and adds nothing to any gradient.

    Returns (q, k), dense, in their dtype; differentiable in q, k and the weights, once and
    in reverse mode (a forward-mode tangent raises; the tables get no gradient)."""
    args = (q, k, q_weight, k_weight, cos, sin, positions)
    _no_tangents("qk_norm_rope", *args[:6])
    if not 0 <= eps < float("inf"):
        raise ValueError(f"eps must be a number not below 0, got {eps}")
    if (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("qk_norm_rope has no gradient for its tables: detach cos and sin")
    rest = float(eps), float(weight_offset), bool(interleaved)
    if not _untraced(*args):
        _rope_sizes(*_call(*args))
        _one_device(*args)
        return qk_norm_rope_op(*args, *rest)
    return (_QkNormRope.apply if grad_needed(*args[:4]) else _forward)(*args, *rest)
