"""What ``fso.ffn`` and ``fso.int4`` refuse, before anything is launched, and the reference that their GPU tests use."""
import ctypes

import pytest
import torch

import ffn_reference as R
import inputs


def _z(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("x,w,kw,text", [
    (_z(4, 16), _z(8, 24), {}, "same K"),
    (_z(4, 16), _z(8), {}, "gate_up"),
    (_z(4, 16), _z(8, 16, dtype=torch.float16), {}, "both"),
    (_z(4, 16, dtype=torch.float32), _z(8, 16, dtype=torch.float32), {}, "both"),
    (_z(4, 16), _z(8, 16), {"activation": "relu"}, "activation"),
    (_z(4, 16), _z(8, 16), {"activation": None}, "activation"),
    (_z(4, 16), _z(8, 16), {}, "CUDA"),
    (torch.tensor(1.0), _z(8, 16), {}, "K"),
    (None, _z(8, 16), {}, "tensor"),
])
def test_gated_linear_refuses(fso, x, w, kw, text):
    with pytest.raises(ValueError, match=text):
        fso.ffn.gated_linear(x, w, **kw)


@pytest.mark.parametrize("codes,scale,zero,text", [
    (_z(4, 64), _z(4, 1), None, "uint8"),
    (_z(4, 64, dtype=torch.uint8), _z(4, 3), None, "power of two"),
    (_z(4, 64, dtype=torch.uint8), _z(4, 8), None, "power of two"),            # groups of 16
    (_z(4, 96, dtype=torch.uint8), _z(4, 2), None, "power of two"),            # groups of 96
    (_z(4, 64, dtype=torch.uint8), _z(3, 1), None, "scale"),
    (_z(4, 64, dtype=torch.uint8), _z(4, 1, dtype=torch.int32), None, "scale"),
    (_z(4, 64, dtype=torch.uint8), _z(4, 1), _z(4, 2, dtype=torch.uint8), "zero"),
    (_z(4, 64, dtype=torch.uint8), _z(4, 1), _z(4, 1), "zero"),
    (_z(0, 64, dtype=torch.uint8), _z(0, 1), None, "codes"),
    (_z(4, 64, dtype=torch.uint8), _z(4, 1), None, "CUDA"),
    (None, _z(4, 1), None, "tensor"),
])
def test_prepare_weight_refuses(fso, codes, scale, zero, text):
    with pytest.raises(ValueError, match=text):
        fso.int4.prepare_weight(codes, scale, zero)


def test_linear_refuses(fso):
    handle = fso.int4.Int4Weight(100, 128, 4, 64, _z(4, 64, dtype=torch.uint8), _z(2, 32), None)
    with pytest.raises(TypeError, match="Int4Weight"):
        fso.int4.linear(_z(2, 128), _z(4, 128))
    for call in (fso.int4.linear, fso.int4.gated_linear):
        with pytest.raises(ValueError, match="in_features"):
            call(_z(2, 120), handle)
        with pytest.raises(ValueError, match="CUDA"):
            call(_z(2, 128), handle)
    with pytest.raises(ValueError, match="activation"):
        fso.int4.gated_linear(_z(2, 128), handle, activation="gelu_erf")
    for kw in ({"group_size": 48}, {"group_size": 512}, {}):
        with pytest.raises(ValueError):
            fso.int4.quantize_weight(_z(4, 512), **kw)


def test_exported_names(fso):
    assert set(fso.ffn.__all__) == {"ACTIVATIONS", "gated_linear"}
    assert set(fso.int4.__all__) == {"ACTIVATIONS", "GROUP_SIZES", "Int4Weight", "prepare_weight", "quantize_weight", "linear",
                                     "gated_linear"}
    assert fso.ffn.ACTIVATIONS == fso.int4.ACTIVATIONS == ("silu", "gelu", "gelu_tanh")
    for name, want in {
        "gated_linear": "(Tensor x, Tensor gate_up, str activation, bool save) -> (Tensor, Tensor)",
        "gated_linear_backward": "(Tensor dh, Tensor x, Tensor gate_up, Tensor saved, str activation, bool need_x, "
                                 "bool need_w) -> (Tensor, Tensor)",
        "int4_linear": "(Tensor x, Tensor codes, Tensor scale, Tensor? zero=None, Tensor? bias=None) -> Tensor",
        "int4_gated_linear": "(Tensor x, Tensor codes, Tensor scale, Tensor? zero, str activation) -> Tensor",
    }.items():
        assert str(getattr(torch.ops.fish_scales_ops, name).default._schema) == f"fish_scales_ops::{name}{want}"


def test_c_entry_points_refuse(fso):
    from fish_scales_ops_b200 import _lib

    L, one, odd = _lib.lib(), ctypes.c_void_p(256), ctypes.c_void_p(264)      # never dereferenced

    def refused(text, name, *args):
        assert getattr(L, name)(*args) == -1 and text in _lib.last_error(), (name, args, _lib.last_error())

    g = "fso_gated_linear"
    refused("multiple of 8", g, one, 16, one, one, None, None, 4, 12, 8, 0, 0, None, 0, None)
    refused("dtype", g, one, 16, one, one, None, None, 4, 16, 8, 2, 0, None, 0, None)
    refused("activation", g, one, 16, one, one, None, None, 4, 16, 8, 0, 3, None, 0, None)
    refused("NULL", g, None, 16, one, one, None, None, 4, 16, 8, 0, 0, None, 0, None)
    refused("go together", g, one, 16, one, one, one, None, 4, 16, 8, 0, 0, None, 0, None)
    refused("ldx", g, one, 20, one, one, None, None, 4, 16, 8, 0, 0, None, 0, None)
    refused("16-byte", g, odd, 16, one, one, None, None, 4, 16, 8, 0, 0, None, 0, None)
    refused("2^24", g, one, 16, one, one, None, None, 1 << 25, 16, 8, 0, 0, None, 0, None)
    b = "fso_gated_linear_backward"
    refused("T > 0", b, one, 8, one, 16, one, one, one, one, one, 0, 16, 8, 0, 0, one, 0, None)
    refused("ldh", b, one, 4, one, 16, one, one, one, one, one, 4, 16, 8, 0, 0, one, 0, None)
    refused("workspace", b, one, 8, one, 16, one, one, one, one, one, 4, 16, 8, 0, 0, one, 0, None)
    i = "fso_int4_linear"
    refused("power of two", i, one, 128, one, one, None, None, one, 4, 8, 128, 48, 0, 0, None)
    refused("power of two", i, one, 128, one, one, None, None, one, 4, 8, 96, 64, 0, 0, None)
    refused("scale_dtype", i, one, 128, one, one, None, None, one, 4, 8, 128, 64, 0, 3, None)
    refused("NULL", i, one, 128, None, one, None, None, one, 4, 8, 128, 64, 0, 0, None)
    refused("16-byte", i, one, 128, odd, one, None, None, one, 4, 8, 128, 64, 0, 0, None)
    refused("activation", "fso_int4_gated_linear", one, 128, one, one, None, one, 4, 8, 128, 64, 0, 0, 5, None)
    refused("group size", "fso_int4_quantize", one, one, one, None, 4, 512, 512, 0, 0, None)
    v = ctypes.c_int64(-1)
    assert L.fso_gated_linear_saved_cols(17, ctypes.byref(v)) == 0 and v.value == 64
    # no rows: nothing to do, whatever the pointers
    assert L.fso_gated_linear(None, 0, None, None, None, None, 0, 16, 8, 0, 0, None, 0, None) == 0
    assert L.fso_int4_linear(None, 0, None, None, None, None, None, 0, 8, 128, 64, 0, 0, None) == 0


@pytest.mark.parametrize("act", R.ACTIVATIONS)
def test_the_reference_gradients_are_differences(act):
    """The 64-bit gradients that the GPU tests compare with, against central differences of the 64-bit projection."""
    x, w, dh = (R.rows(*s, seed, torch.float64) for seed, s in enumerate(((5, 16), (14, 16), (5, 7))))
    dx, _, dw, _ = R.gated_backward(x, w, act, dh)
    g = x @ w.t()
    a, s = R.act_and_slope(g, act)
    e = 1e-5
    up, down = R.act_and_slope(g + e, act)[0], R.act_and_slope(g - e, act)[0]
    assert torch.allclose((up - down) / (2 * e), s, atol=1e-8, rtol=1e-6)
    f = lambda p, q: float(((R.act_and_slope(p @ q[:7].t(), act)[0] * (p @ q[7:].t())) * dh).sum())  # noqa: E731
    for seed in range(4):
        v, u = (torch.randn(m.shape, generator=inputs.gen(seed), dtype=torch.float64) for m in (x, w))
        assert abs((f(x + e * v, w) - f(x - e * v, w)) / (2 * e) - float((dx * v).sum())) < 1e-5
        assert abs((f(x, w + e * u) - f(x, w - e * u)) / (2 * e) - float((dw * u).sum())) < 1e-5


def test_two_codes_in_a_byte():
    codes = torch.tensor([[0x21, 0x43]], dtype=torch.uint8)
    assert R.unpack(codes).tolist() == [[1, 2, 3, 4]]
    w = R.dequantize(codes.repeat(1, 8), torch.tensor([[2.0]]), torch.tensor([[3]], dtype=torch.uint8))
    assert w[0, :4].tolist() == [-4.0, -2.0, 0.0, 2.0]
