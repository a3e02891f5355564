"""``fso.ffn`` on a B200: the gated feed-forward projection in 16 bits, forward and backward.

    h = fso.ffn.gated_linear(x, gate_up, activation="silu")     # act(x G^T) * (x U^T), differentiable

``gate_up [2*INTER, K]`` stacks the gate rows G over the up rows U, the order of ``fso.compat.prepare_gate_up`` and of
checkpoints. ``fso.compat.linear_swiglu`` is the MXFP8 form of the same step (forward only), ``fso.int4.gated_linear`` the
one over 4-bit weights for decode. One tcgen05 kernel computes both projections, the activation and their product; its
gradients are two more products of the same kernel family. The reference has no counterpart.

Errors are those of the other namespaces: ValueError for a malformed argument, NotImplementedError for what is not
served, raised before anything is launched.
"""
import torch

from .. import _ops
from .._arch import SERVED_MAJOR, arch_label, device_arch

__all__ = ["ACTIVATIONS", "gated_linear"]

ACTIVATIONS = tuple(_ops.GATE_ACTIVATIONS)
_MAX_DIM = 1 << 24


def _check(op: str, x, gate_up, activation) -> None:
    """``op``: the name in a refusal, which begins with the device's."""
    if activation not in _ops.GATE_ACTIVATIONS:
        _refuse(op, f"unknown activation {activation!r}; the activations are {', '.join(ACTIVATIONS)}")
    if x.dim() != 2 or gate_up.dim() != 2 or x.shape[1] != gate_up.shape[1]:
        _refuse(op, f"x must be [..., K] and gate_up [2*INTER, K] with the same K, got {tuple(x.shape)} and "
                    f"{tuple(gate_up.shape)}")
    if x.dtype not in _ops.DTYPES_16 or gate_up.dtype != x.dtype:
        _refuse(op, f"x and gate_up must both be bf16 or both fp16, got {x.dtype} and {gate_up.dtype}")
    if not x.is_cuda or gate_up.get_device() != x.get_device():
        _refuse(op, f"x and gate_up must be on one CUDA device, got {x.device} and {gate_up.device}")
    rows, k = gate_up.shape
    if rows < 2 or rows % 2 != 0 or k < 8 or k % 8 != 0:
        _refuse(op, f"gate_up must have an even number of rows and K a positive multiple of 8, got {tuple(gate_up.shape)}")
    if rows // 2 > _MAX_DIM or k > _MAX_DIM or x.shape[0] > _MAX_DIM:
        _refuse(op, f"a dimension of {tuple(x.shape)} or {tuple(gate_up.shape)} is beyond 2^24")
    if not gate_up.is_contiguous() or gate_up.data_ptr() % 16 != 0:
        _refuse(op, f"gate_up must be contiguous and start on a 16-byte boundary (it is read in place with TMA), got strides "
                    f"{tuple(gate_up.stride())}")
    if device_arch() // 10 != SERVED_MAJOR:
        raise NotImplementedError(f"{op} ({arch_label(device_arch())}): this build serves sm_100-family devices")


def _refuse(op: str, why: str):
    raise ValueError(f"{op} ({arch_label(device_arch())}): {why}")


# ------------------------------------------------------------------------------------------------ custom ops

def _gated_linear_body(x, gate_up, activation, save):
    _check("fish_scales_ops::gated_linear", x, gate_up, activation)
    h, saved = _ops.gated_linear(x, gate_up, _ops.GATE_ACTIVATIONS[activation], save)
    return h, saved if save else x.new_empty((x.shape[0], 0), dtype=torch.uint8)


def _gated_linear_backward_body(dh, x, gate_up, saved, activation, need_x, need_w):
    op = "fish_scales_ops::gated_linear_backward"
    _check(op, x, gate_up, activation)
    t, inter = int(x.shape[0]), int(gate_up.shape[0]) // 2
    cols = _ops.gated_saved_cols(inter)
    if tuple(dh.shape) != (t, inter) or dh.dtype != x.dtype or dh.device != x.device:
        _refuse(op, f"dh must be {x.dtype} [{t}, {inter}] on {x.device}, got {dh.dtype} {tuple(dh.shape)} on {dh.device}")
    if tuple(saved.shape) != (t, cols) or saved.dtype != torch.uint8 or saved.device != x.device or not saved.is_contiguous():
        _refuse(op, f"saved must be the uint8 [{t}, {cols}] that fish_scales_ops::gated_linear returned with save, got "
                    f"{saved.dtype} {tuple(saved.shape)}")
    dx, dw = _ops.gated_linear_backward(dh, x, gate_up, saved, _ops.GATE_ACTIVATIONS[activation], need_x, need_w)
    empty = x.new_empty((0, x.shape[1]))
    return dx if need_x else empty, dw if need_w else empty


_gated_linear_op = torch.library.custom_op(
    "fish_scales_ops::gated_linear",
    mutates_args=(),
    schema="(Tensor x, Tensor gate_up, str activation, bool save) -> (Tensor, Tensor)",
)(_gated_linear_body)

_gated_linear_backward_op = torch.library.custom_op(
    "fish_scales_ops::gated_linear_backward",
    mutates_args=(),
    schema="(Tensor dh, Tensor x, Tensor gate_up, Tensor saved, str activation, bool need_x, bool need_w) "
           "-> (Tensor, Tensor)",
)(_gated_linear_backward_body)


@_gated_linear_op.register_fake
def _gated_linear_fake(x, gate_up, activation, save):
    t, inter = x.shape[0], gate_up.shape[0] // 2
    return x.new_empty((t, inter)), x.new_empty((t, 6 * ((inter + 15) // 16 * 16) if save else 0), dtype=torch.uint8)


@_gated_linear_backward_op.register_fake
def _gated_linear_backward_fake(dh, x, gate_up, saved, activation, need_x, need_w):
    return (x.new_empty((x.shape[0] if need_x else 0, x.shape[1])),
            x.new_empty((gate_up.shape[0] if need_w else 0, x.shape[1])))


def _setup_context(ctx, inputs, output):
    x, gate_up, activation, save = inputs
    if not save:
        raise RuntimeError("fish_scales_ops::gated_linear: a gradient needs what save=True keeps")
    ctx.save_for_backward(x, gate_up, output[1])
    ctx.activation = activation
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _op_backward(ctx, dh, *_):
    x, gate_up, saved = ctx.saved_tensors
    need_x, need_w = ctx.needs_input_grad[:2]
    if dh is None or not (need_x or need_w):
        return None, None, None, None
    dx, dw = torch.ops.fish_scales_ops.gated_linear_backward(dh, x, gate_up, saved, ctx.activation, need_x, need_w)
    return dx if need_x else None, dw if need_w else None, None, None


_gated_linear_op.register_autograd(_op_backward, setup_context=_setup_context)


class _GatedLinear(torch.autograd.Function):
    """The eager form: the kernels behind the two custom ops, without the dispatcher's round trip and with the checks made
    once."""

    @staticmethod
    def forward(ctx, x, gate_up, activation):
        _check("fso.ffn.gated_linear", x, gate_up, activation)
        act = _ops.GATE_ACTIVATIONS[activation]
        h, saved = _ops.gated_linear(x, gate_up, act, True)
        ctx.save_for_backward(x, gate_up, saved)
        ctx.act = act
        return h

    @staticmethod
    def backward(ctx, dh):
        if torch.is_grad_enabled():      # create_graph: the gradients come with a node that refuses to be differentiated
            return _differentiable_once(ctx, dh)
        return _eager_backward(ctx, dh)


def _eager_backward(ctx, dh):
    x, gate_up, saved = ctx.saved_tensors
    need_x, need_w, _ = ctx.needs_input_grad
    dx, dw = _ops.gated_linear_backward(dh, x, gate_up, saved, ctx.act, need_x, need_w)
    return dx, dw, None


_differentiable_once = torch.autograd.function.once_differentiable(_eager_backward)


# ------------------------------------------------------------------------------------------------ public functions

def gated_linear(x: torch.Tensor, gate_up: torch.Tensor, *, activation: str = "silu") -> torch.Tensor:
    """``act(x G^T) * (x U^T)``: ``x [..., K]``, ``gate_up [2*INTER, K]`` with the gate rows first, both bf16 or both fp16;
    returns ``[..., INTER]`` of the same type. ``activation``: ``"silu"``, ``"gelu"`` (erf) or ``"gelu_tanh"``.
    ``K % 8 == 0``; INTER and the number of rows are free (no row at all included). ``x`` may be a slice of wider rows (it
    is read in place when its rows start on 16-byte boundaries and copied otherwise); ``gate_up`` must be contiguous.

    Sums are fp32, the result is rounded once. Differentiable in both arguments, once: where a gradient is wanted the call
    keeps the projections in 24 bits (6 bytes for each value of the result), the backward pass rounds the
    gradients of the projections to the 16-bit type and multiplies them with gate_up and x; where none is wanted
    nothing is kept. The same bits come out of the same call every time. Nothing synchronizes; the call and its backward pass
    can be captured into a CUDA graph after one eager call of the same shape, provided that no eager graph of the same
    leaves is alive then (torch cannot capture a backward pass otherwise)."""
    if not isinstance(x, torch.Tensor) or not isinstance(gate_up, torch.Tensor) or x.dim() < 1:
        raise ValueError("fso.ffn.gated_linear: x must be a [..., K] and gate_up a [2*INTER, K] tensor")
    lead = x.shape[:-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1]) if x.shape[-1] > 0 else x.new_empty((0, 0))
    grad = torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad)
    if torch.compiler.is_compiling():
        h = torch.ops.fish_scales_ops.gated_linear(x2, gate_up, activation, grad)[0]
    elif grad:
        h = _GatedLinear.apply(x2, gate_up, activation)
    else:
        _check("fso.ffn.gated_linear", x2, gate_up, activation)
        h = _ops.gated_linear(x2, gate_up, _ops.GATE_ACTIVATIONS[activation], False)[0]
    return h if x.dim() == 2 else h.reshape(*lead, h.shape[1])
