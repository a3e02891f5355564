"""``fso.int4`` on a B200: linear layers over 4-bit weights with group scales, for the few rows of a decode step.

    weight = fso.int4.prepare_weight(codes, scale, zero)         # a checkpoint's codes, scales and zero points
    weight = fso.int4.quantize_weight(w, group_size=128)         # or a 16-bit weight, rounded to the nearest step
    y = fso.int4.linear(x, weight)                               # x W^T
    h = fso.int4.gated_linear(x, gate_up, activation="silu")     # act(x G^T) * (x U^T) in one kernel

``W[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group])`` with codes 0..15, two in a byte (even k in the
lower four bits). The activations stay in 16 bits. ``fso.dense`` holds the 8-bit formats, which suit many rows;
``fso.ffn.gated_linear`` is the gated projection in 16 bits, with gradients. The reference has no counterpart.

Forward only. Errors are those of the other namespaces: ValueError for a malformed argument, NotImplementedError for
what is not served, TypeError for a wrong handle, raised before anything is launched.
"""
import dataclasses
from typing import Optional

import torch

from .. import _ops
from .._arch import SERVED_MAJOR, arch_label, device_arch

__all__ = ["ACTIVATIONS", "GROUP_SIZES", "Int4Weight", "prepare_weight", "quantize_weight", "linear", "gated_linear"]

ACTIVATIONS = tuple(_ops.GATE_ACTIVATIONS)
GROUP_SIZES = (32, 64, 128, 256)       # of quantize_weight; prepare_weight takes any larger power of two as well
_SCALE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_MAX_DIM = 1 << 24
_MAX_ROWS = 65535 * 64


def _by_halves(t: torch.Tensor) -> torch.Tensor:
    """[N, groups] -> [groups, 2 * half], the layout the kernels read; columns between the halves are zero."""
    n, first, half = t.shape[0], (t.shape[0] + 1) // 2, _ops.int4_half_cols(t.shape[0])
    if n == 2 * half:
        return t.t().clone(memory_format=torch.contiguous_format)      # never the caller's memory
    out = t.new_zeros((t.shape[1], 2 * half))
    out[:, :first].copy_(t[:first].t())
    out[:, half:half + n - first].copy_(t[first:].t())
    return out


def _rows_of(t: torch.Tensor, n: int) -> torch.Tensor:
    """The inverse of :func:`_by_halves`."""
    first, half = (n + 1) // 2, t.shape[1] // 2
    return torch.cat((t[:, :first], t[:, half:half + n - first]), 1).t()


@dataclasses.dataclass(frozen=True, eq=False, repr=False)
class Int4Weight:
    """One 4-bit weight: ``codes`` uint8 ``[N, K/2]``, ``scale`` bf16, fp16 or fp32 ``[N, K/group_size]``, ``zero`` uint8
    of the same shape or None (8 everywhere), as a checkpoint stores them. What the kernels read is ``packed``, the codes with
    the even k of every eight in the lower four nibbles of a 32-bit word and the odd k in the upper four, and ``scale_t``
    and ``zero_t`` ``[K/group_size, 2 * half]``, transposed and by halves of the rows: ``half`` is half of N rounded up to a
    multiple of 16, the first half of the rows starts at column 0 and the second at column ``half``. ``codes``, ``scale`` and
    ``zero`` are made of them when asked for.

    A call starts to load the weight before the kernel ahead of it on the stream has finished. Whoever rewrites a handle's
    tensors in place has a kernel that does not write them run between that and the next call (the functions that make a
    handle see to it themselves)."""

    arch: int
    in_features: int
    out_features: int
    group_size: int
    packed: torch.Tensor
    scale_t: torch.Tensor
    zero_t: Optional[torch.Tensor]

    @property
    def codes(self) -> torch.Tensor:
        b = self.packed.view(self.out_features, -1, 4)      # bytes: k 0 2, 4 6, 1 3, 5 7
        even = torch.stack((b[..., 0] & 15, b[..., 0] >> 4, b[..., 1] & 15, b[..., 1] >> 4), -1)
        odd = torch.stack((b[..., 2] & 15, b[..., 2] >> 4, b[..., 3] & 15, b[..., 3] >> 4), -1)
        return (even | (odd << 4)).flatten(1)

    @property
    def scale(self) -> torch.Tensor:
        return _rows_of(self.scale_t, self.out_features)

    @property
    def zero(self) -> Optional[torch.Tensor]:
        return None if self.zero_t is None else _rows_of(self.zero_t, self.out_features)

    def __repr__(self) -> str:
        return (f"Int4Weight(arch=sm_{self.arch}, in_features={self.in_features}, out_features={self.out_features}, "
                f"group_size={self.group_size}, scale={self.scale_t.dtype}, zero={'none' if self.zero_t is None else 'uint8'})")


def _check_weight(op: str, codes, scale, zero) -> None:
    """The three tensors of a weight as the kernels read them, by their metadata alone."""
    if codes.dtype != torch.uint8 or codes.dim() != 2 or codes.shape[0] < 1 or codes.shape[1] < 16:
        raise ValueError(f"{op}: codes must be a uint8 [N, K/2] tensor, two codes in a byte, got {codes.dtype} "
                         f"{tuple(codes.shape)}")
    n, k = int(codes.shape[0]), 2 * int(codes.shape[1])
    cols = 2 * _ops.int4_half_cols(n)
    if scale.dtype not in _SCALE_DTYPES or scale.dim() != 2 or scale.shape[1] != cols or scale.shape[0] < 1:
        raise ValueError(f"{op}: scale must be bf16, fp16 or fp32 [K/group, {cols}] for {n} rows (the layout of "
                         f"fso.int4.Int4Weight.scale_t), got {scale.dtype} {tuple(scale.shape)}")
    groups = int(scale.shape[0])
    group = k // groups
    if group * groups != k or group < 32 or group & (group - 1):
        raise ValueError(f"{op}: {groups} scales for a row of K = {k}: the group size must be a power of two of at least 32 "
                         f"that divides K")
    if zero is not None and (zero.dtype != torch.uint8 or zero.shape != scale.shape):
        raise ValueError(f"{op}: zero must be uint8 and shaped like scale, got {zero.dtype} {tuple(zero.shape)} for "
                         f"{tuple(scale.shape)}")
    if n > _MAX_DIM or k > _MAX_DIM:
        raise ValueError(f"{op}: a dimension of [{n}, {k}] is beyond 2^24")
    for name, t in (("codes", codes), ("scale", scale), ("zero", zero)):
        if t is None:
            continue
        if not t.is_cuda or t.device != codes.device:
            raise ValueError(f"{op}: codes, scale and zero must be on one CUDA device, {name} is on {t.device}")
        if not t.is_contiguous() or t.data_ptr() % 16 != 0:
            raise ValueError(f"{op}: {name} must be contiguous and start on a 16-byte boundary, got strides "
                             f"{tuple(t.stride())}; fso.int4.prepare_weight returns such tensors")


def _check_x(op: str, x, codes) -> None:
    k = 2 * codes.shape[1]
    if x.dim() != 2 or x.shape[1] != k:
        raise ValueError(f"{op}: x must be [..., {k}] (K = in_features), got {tuple(x.shape)}")
    if x.dtype not in _ops.DTYPES_16:
        raise ValueError(f"{op}: x must be bf16 or fp16, got {x.dtype}")
    if not x.is_cuda or x.get_device() != codes.get_device():
        raise ValueError(f"{op}: x lives on {x.device}, the weight on {codes.device}; both must be on one CUDA device")
    if x.shape[0] > _MAX_ROWS:
        raise ValueError(f"{op}: {int(x.shape[0])} rows of x; at most {_MAX_ROWS} are served")


def _check_bias(op: str, bias, x, n: int) -> None:
    if bias.dtype != x.dtype or tuple(bias.shape) != (n,) or bias.device != x.device or not bias.is_contiguous():
        raise ValueError(f"{op}: bias must be a contiguous {x.dtype} [{n}] tensor on {x.device}, got {bias.dtype} "
                         f"{tuple(bias.shape)} on {bias.device}")


def _check_gate(op: str, codes, activation) -> None:
    if activation not in _ops.GATE_ACTIVATIONS:
        raise ValueError(f"{op}: unknown activation {activation!r}; the activations are {', '.join(ACTIVATIONS)}")
    if codes.shape[0] % 2 != 0:
        raise ValueError(f"{op}: a gate_up weight has an even number of rows, got {int(codes.shape[0])}")


def _need_arch(op: str) -> None:
    if device_arch() // 10 != SERVED_MAJOR:
        raise NotImplementedError(f"{op}: this build serves sm_100-family devices")


def _complete(handle: Int4Weight) -> Int4Weight:
    """One empty plain launch behind whatever wrote the handle's tensors: a call on it starts to load the weight before
    its predecessor on the stream has finished, which is only safe when that predecessor did not write it."""
    _ops.stream_fence(handle.packed.device)
    return handle


def _aligned(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# ------------------------------------------------------------------------------------------------ custom ops

# The ops check all their tensors. The public functions below check a handle's tensors when they make the handle, not at
# each call: the checks would take longer than a decode-sized kernel runs.

def _int4_linear_body(x, codes, scale, zero=None, bias=None):
    op = f"fish_scales_ops::int4_linear ({arch_label(device_arch())})"
    _check_weight(op, codes, scale, zero)
    _check_x(op, x, codes)
    if bias is not None:
        _check_bias(op, bias, x, int(codes.shape[0]))
    _need_arch(op)
    return _ops.int4_linear(x, codes, scale, zero, bias)


def _int4_gated_linear_body(x, codes, scale, zero, activation):
    op = f"fish_scales_ops::int4_gated_linear ({arch_label(device_arch())})"
    _check_weight(op, codes, scale, zero)
    _check_gate(op, codes, activation)
    _check_x(op, x, codes)
    _need_arch(op)
    return _ops.int4_gated_linear(x, codes, scale, zero, _ops.GATE_ACTIVATIONS[activation])


_int4_linear_op = torch.library.custom_op(
    "fish_scales_ops::int4_linear",
    mutates_args=(),
    schema="(Tensor x, Tensor codes, Tensor scale, Tensor? zero=None, Tensor? bias=None) -> Tensor",
)(_int4_linear_body)

_int4_gated_linear_op = torch.library.custom_op(
    "fish_scales_ops::int4_gated_linear",
    mutates_args=(),
    schema="(Tensor x, Tensor codes, Tensor scale, Tensor? zero, str activation) -> Tensor",
)(_int4_gated_linear_body)


@_int4_linear_op.register_fake
def _int4_linear_fake(x, codes, scale, zero=None, bias=None):
    return x.new_empty((x.shape[0], codes.shape[0]))


@_int4_gated_linear_op.register_fake
def _int4_gated_linear_fake(x, codes, scale, zero, activation):
    return x.new_empty((x.shape[0], codes.shape[0] // 2))


# ------------------------------------------------------------------------------------------------ public functions

def prepare_weight(codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None) -> Int4Weight:
    """The handle of a weight that a checkpoint stores in 4 bits: ``codes`` uint8 ``[N, K/2]``, ``scale`` bf16, fp16 or
    fp32 ``[N, K/group]``, ``zero`` uint8 ``[N, K/group]`` with values 0..15 (None: 8 everywhere). The group size is a power
    of two of at least 32. All three are laid out anew for the kernels (one pass over each). The values of ``zero`` are not
    looked at (that would synchronize)."""
    ctx = "fso.int4.prepare_weight"
    for name, t in (("codes", codes), ("scale", scale), ("zero", zero)):
        if not isinstance(t, torch.Tensor) and not (name == "zero" and t is None):
            raise ValueError(f"{ctx}: {name} must be a tensor, got {type(t).__name__}")
    for name, t in (("scale", scale), ("zero", zero)):
        if t is not None and (t.dim() != 2 or codes.dim() < 1 or t.shape[0] != codes.shape[0] or 0 in t.shape):
            raise ValueError(f"{ctx}: {name} must be a [N, K/group] tensor for the codes' {codes.shape[0]} rows, got "
                             f"{tuple(t.shape)}")
    codes, scale_t = _aligned(codes.detach()), _by_halves(scale.detach())
    zero_t = None if zero is None else _by_halves(zero.detach())
    _check_weight(ctx, codes, scale_t, zero_t)
    _need_arch(ctx)
    k = 2 * int(codes.shape[1])
    return _complete(Int4Weight(device_arch(), k, int(codes.shape[0]), k // int(scale_t.shape[0]), _ops.int4_pack_codes(codes),
                                scale_t, zero_t))


def quantize_weight(w: torch.Tensor, *, group_size: int = 128, zero_point: bool = False,
                    scale_dtype: Optional[torch.dtype] = None) -> Int4Weight:
    """A bf16 or fp16 weight ``[N, K]`` rounded to 4 bits, each group by itself and to the nearest step. Without
    ``zero_point`` the step is ``amax / 7`` and codes run from 1 to 15 around 8; with it the step is ``(hi - lo) / 15``
    for the group's range with zero inside, and the zero point ``round(-lo / step)``. The step is rounded to
    ``scale_dtype`` (default: the weight's type) before the codes are taken. ``group_size`` is one of 32, 64, 128, 256
    and divides K. A group that holds a NaN or an infinity gets a scale that is not a number."""
    ctx = "fso.int4.quantize_weight"
    if not isinstance(w, torch.Tensor) or w.dim() != 2 or w.dtype not in _ops.DTYPES_16 or not w.is_cuda:
        raise ValueError(f"{ctx}: w must be a CUDA bf16 or fp16 [N, K] tensor")
    if group_size not in GROUP_SIZES or int(w.shape[1]) % group_size != 0 or 0 in w.shape:
        raise ValueError(f"{ctx}: group_size must be one of {GROUP_SIZES} and divide K, got {group_size} for "
                         f"{tuple(w.shape)}")
    if max(w.shape) > _MAX_DIM:
        raise ValueError(f"{ctx}: a dimension of {tuple(w.shape)} is beyond 2^24")
    scale_dtype = w.dtype if scale_dtype is None else scale_dtype
    if scale_dtype not in _SCALE_DTYPES:
        raise ValueError(f"{ctx}: scale_dtype must be bf16, fp16 or fp32, got {scale_dtype}")
    _need_arch(ctx)
    codes, scale, zero = _ops.int4_quantize(_aligned(w.detach()), group_size, bool(zero_point), scale_dtype)
    return _complete(Int4Weight(device_arch(), int(w.shape[1]), int(w.shape[0]), int(group_size), codes, scale, zero))


def _flatten(x, weight, ctx: str):
    if not isinstance(weight, Int4Weight):
        raise TypeError(f"{ctx}: the weight argument is a {type(weight).__name__}; pass the Int4Weight that "
                        f"fso.int4.prepare_weight or fso.int4.quantize_weight returned")
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] != weight.in_features:
        shown = tuple(x.shape) if isinstance(x, torch.Tensor) else type(x).__name__
        raise ValueError(f"{ctx}: x must be [..., {weight.in_features}] (K = in_features), got {shown}")
    return x if x.dim() == 2 else x.reshape(-1, weight.in_features)


def linear(x: torch.Tensor, weight: Int4Weight, *, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x W^T (+ bias)``: ``x [..., K]`` bf16 or fp16, result ``[..., N]`` of the same type; ``bias [N]`` of the same type is
    added before the one rounding. ``x`` may be a slice of wider rows. The products are exact, sums and scales fp32, and
    the same bits come out of the same call every time. Any number of rows is served, none included; the kernel is made
    for the few of a decode step. Nothing synchronizes; the call can be captured into a CUDA graph after one eager call
    of the same shape."""
    x2 = _flatten(x, weight, "fso.int4.linear")
    if torch.compiler.is_compiling():
        y = torch.ops.fish_scales_ops.int4_linear(x2, weight.packed, weight.scale_t, weight.zero_t, bias)
    else:
        _check_x("fso.int4.linear", x2, weight.packed)
        if bias is not None:
            _check_bias("fso.int4.linear", bias, x2, weight.out_features)
        y = _ops.int4_linear(x2, weight.packed, weight.scale_t, weight.zero_t, bias)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], weight.out_features)


def gated_linear(x: torch.Tensor, gate_up: Int4Weight, *, activation: str = "silu") -> torch.Tensor:
    """``act(x G^T) * (x U^T)`` in one kernel, G the first and U the last half of the rows of ``gate_up`` (the order of
    ``fso.ffn.gated_linear``): ``x [..., K]`` bf16 or fp16, result ``[..., N/2]`` of the same type. ``activation``:
    ``"silu"``, ``"gelu"`` (erf) or ``"gelu_tanh"``. Otherwise as :func:`linear`."""
    x2 = _flatten(x, gate_up, "fso.int4.gated_linear")
    if torch.compiler.is_compiling():
        h = torch.ops.fish_scales_ops.int4_gated_linear(x2, gate_up.packed, gate_up.scale_t, gate_up.zero_t, activation)
    else:
        _check_gate("fso.int4.gated_linear", gate_up.packed, activation)
        _check_x("fso.int4.gated_linear", x2, gate_up.packed)
        h = _ops.int4_gated_linear(x2, gate_up.packed, gate_up.scale_t, gate_up.zero_t, _ops.GATE_ACTIVATIONS[activation])
    return h if x.dim() == 2 else h.reshape(*x.shape[:-1], gate_up.out_features // 2)
