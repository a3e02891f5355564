"""``fso.ffn.gated_linear`` and its gradients against the definition in 64 bits, element by element within the bound that
fp32 sums and the stated roundings allow (ffn_reference), at sizes around the tiles (256 x 128, 64 of the contraction)."""
import pytest
import torch

import ffn_reference as R
import inputs

pytestmark = pytest.mark.gpu

SIZES = [(1, 8, 1), (1, 64, 128), (3, 72, 17), (16, 4096, 40), (17, 520, 300), (64, 128, 64), (65, 264, 65), (100, 2048, 33),
         (128, 256, 256), (129, 1032, 130), (257, 64, 129), (300, 200, 1000), (513, 136, 264), (1030, 72, 520)]
SPLIT = [(512, 7168, 256), (500, 7168, 251), (260, 4104, 24)]      # few tiles, long contractions: sums of slices


def _case(t, k, i, dtype, seed=0):
    x = R.rows(t, k, seed + 1, dtype)
    w = R.rows(2 * i, k, seed + 2, dtype, std=k ** -0.5)
    return x.cuda(), w.cuda(), R.rows(t, i, seed + 3, dtype).cuda()


def _grads(fso, x, w, dh, act):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    h = fso.ffn.gated_linear(x, w, activation=act)
    return (h.detach(), *torch.autograd.grad(h, (x, w), dh))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("t,k,i", SIZES + SPLIT)
def test_forward_and_gradients(fso, device_ok, t, k, i, dtype):
    act = R.ACTIVATIONS[(t + i) % 3]
    x, w, dh = _case(t, k, i, dtype)
    h, bound, _, _ = R.gated(x, w, act)
    with torch.no_grad():
        R.inside(fso.ffn.gated_linear(x, w, activation=act), h, bound, "h")
    got, dx, dw = _grads(fso, x, w, dh, act)
    assert dx.shape == x.shape and dw.shape == w.shape and dx.dtype == dw.dtype == dtype
    R.inside(got, h, bound, "h with saved projections")
    wx, bx, ww, bw = R.gated_backward(x, w, act, dh)
    R.inside(dx, wx, bx, "dx")
    R.inside(dw, ww, bw, "dgate_up")
    # the roundings of the terms of a sum are independent: together, over many values, less than two half steps
    if t * k > 4096 and i > 32:
        for g, want in ((dx, wx), (dw, ww)):
            assert inputs.rel_frobenius(g.double().cpu(), want.cpu()) <= 2 * R.half_step(dtype)


@pytest.mark.parametrize("act", R.ACTIVATIONS)
def test_gradients_against_differences(fso, device_ok, act):
    """Along random directions: (f(x + e v) - f(x - e v)) / 2e of f = sum(h dh) in 64 bits, where neither the differences
    (e^2) nor 64 bits are seen; the kernel's gradient may be off by its own bound times |v|."""
    x, w, dh = _case(37, 128, 96, torch.bfloat16, 5)
    _, dx, dw = _grads(fso, x, w, dh, act)
    _, bx, _, bw = R.gated_backward(x, w, act, dh)
    f = lambda a, b: float((R.gated(a, b, act)[0] * dh.double()).sum())  # noqa: E731
    xd, wd, e = x.double(), w.double(), 1e-4
    R_x = lambda d: f(xd + d, wd)  # noqa: E731
    R_w = lambda d: f(xd, wd + d)  # noqa: E731
    for val, g, b, at in ((xd, dx, bx, R_x), (wd, dw, bw, R_w)):
        for seed in range(3):
            v = torch.randn(val.shape, generator=inputs.gen(seed), dtype=torch.float64).cuda()
            diff = (at(e * v) - at(-e * v)) / (2 * e)
            assert abs(float((g.double() * v).sum()) - diff) <= float((b * v.abs()).sum()) + 1e-6 * abs(diff)


def test_rows_are_read_where_they_lie(fso, device_ok):
    """Slices of wider rows, rows off a 16-byte boundary, every second row, one row for all, leading dimensions: the bits of
    the same rows laid out densely, and gradients of the shape that came in."""
    k, i, t = 200, 72, 40
    buf = R.rows(2 * t, k + 40, 1, torch.bfloat16).cuda()
    w = R.rows(2 * i, k, 2, torch.bfloat16, std=0.07).cuda()
    views = {"slice": buf[:t, 8:8 + k], "off the boundary": buf[:t, 3:3 + k], "every second row": buf[::2, :k],
             "expanded": buf[5:6, :k].expand(t, k), "columns apart": buf[:t].t().contiguous().t()[:, :k],
             "three dimensions": buf[:, :k].view(2, t, k)}
    for name, x in views.items():
        dense = x.contiguous()
        x1, x2 = x.detach().requires_grad_(), dense.detach().requires_grad_()
        h1, h2 = fso.ffn.gated_linear(x1, w), fso.ffn.gated_linear(x2, w)
        assert h1.shape == x.shape[:-1] + (i,) and torch.equal(h1, h2), name
        dh = torch.randn_like(h1)
        g1, g2 = torch.autograd.grad(h1, x1, dh)[0], torch.autograd.grad(h2, x2, dh)[0]
        assert g1.shape == x.shape and torch.equal(g1, g2), name


def test_gradient_layouts_and_single_gradients(fso, device_ok):
    """dh broadcast by a sum, dh with strides, one of the two gradients alone: the bits of the dense, complete call."""
    x, w, dh = _case(50, 136, 88, torch.float16)
    _, dx, dw = _grads(fso, x, w, dh, "silu")
    strided = torch.empty(50, 88 * 3, dtype=dh.dtype, device="cuda")[:, 5:93]
    strided.copy_(dh)
    for d in (strided, dh.t().contiguous().t()):
        _, gx, gw = _grads(fso, x, w, d, "silu")
        assert torch.equal(gx, dx) and torch.equal(gw, dw)
    _, ox, ow = _grads(fso, x, w, torch.ones_like(dh), "silu")
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    fso.ffn.gated_linear(xr, wr).sum().backward()
    assert torch.equal(xr.grad, ox) and torch.equal(wr.grad, ow)
    only_x, only_w = x.detach().requires_grad_(), w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(fso.ffn.gated_linear(only_x, w), only_x, dh)[0], dx)
    assert torch.equal(torch.autograd.grad(fso.ffn.gated_linear(x, only_w), only_w, dh)[0], dw)


def test_no_rows(fso, device_ok):
    w = R.rows(20, 16, 1, torch.bfloat16).cuda().requires_grad_()
    for shape in ((0, 16), (3, 0, 16)):
        x = torch.empty(shape, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        h = fso.ffn.gated_linear(x, w)
        assert h.shape == shape[:-1] + (10,)
        dx, dw = torch.autograd.grad(h.sum(), (x, w))
        assert dx.shape == x.shape and not dw.any() and dw.shape == w.shape


def test_extreme_values_stay_in_their_row(fso, device_ok):
    """A NaN, an infinity and large finite values in single rows: other rows keep their bits, large gates saturate."""
    x, w, dh = _case(140, 64, 40, torch.bfloat16)
    want, wdx, _ = _grads(fso, x, w, dh, "silu")
    y = x.clone()
    y[3, 5] = float("nan")
    y[130, 0] = float("inf")
    y[7] *= 1e4
    h, dx, _ = _grads(fso, y, w, dh, "silu")
    keep = torch.ones(140, dtype=torch.bool, device="cuda")
    keep[[3, 7, 130]] = False
    assert torch.equal(h[keep], want[keep]) and torch.equal(dx[keep], wdx[keep])
    assert torch.isnan(h[3]).all() and torch.isnan(dx[3]).all() and not torch.isfinite(h[130]).any()
    for act in R.ACTIVATIONS:
        big, bound, _, _ = R.gated(y[7:8], w, act)
        R.inside(fso.ffn.gated_linear(y[7:8], w, activation=act), big, bound, act)
        assert torch.isfinite(torch.cat(_grads(fso, y[7:8], w, dh[7:8], act)[:2], 1)).all()


@pytest.mark.parametrize("act", R.ACTIVATIONS)
def test_gates_of_any_finite_size(fso, device_ok, act):
    """Gates up to 1e30, whose squares fp32 does not hold: there act(g) is g or 0 and its slope 1 or 0. dg and du are rounded
    once and so is their sum, g and u are in 24 bits, and 1e-5 is for the activation's own arithmetic."""
    x = torch.tensor([[s * 10.0 ** e] + [0.0] * 7 for e in (5, 13, 19, 20, 30) for s in (1, -1)], dtype=torch.bfloat16).cuda()
    w = torch.zeros(2, 8, dtype=torch.bfloat16, device="cuda")
    w[0, 0], w[1, 0] = 1.0, 2.0 ** -100      # g = x, u = 2^-100 x
    dh = torch.full((10, 1), 2.0 ** -20, dtype=torch.bfloat16, device="cuda")
    xr = x.detach().requires_grad_()
    h = fso.ffn.gated_linear(xr, w, activation=act)
    (dx,) = torch.autograd.grad(h, xr, dh)
    g = x[:, 0].double().clamp(min=0)
    want, slope = g * g * 2.0 ** -100, 2 * g * 2.0 ** -120
    he = R.half_step(torch.bfloat16)
    assert ((h[:, 0].double() - want).abs() <= (he + 1e-5) * want).all()
    assert ((dx[:, 0].double() - slope).abs() <= (2 * he + he * he + 2.0 ** -14 + 1e-5) * slope).all()


def test_same_bits_every_time_and_on_another_stream(fso, device_ok):
    x, w, dh = _case(700, 264, 300, torch.bfloat16)
    first = _grads(fso, x, w, dh, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _grads(fso, x, w, dh, "gelu")
    side.synchronize()
    for a, b, c in zip(first, other, _grads(fso, x, w, dh, "gelu")):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_steps_beside_an_eager_graph(fso, device_ok):
    """Two captured training steps of different sizes, replayed in turn with new inputs while an eager graph over the same
    memory is alive: each gives the eager call's bits. (The eager graph has leaves of its own: torch cannot capture a
    backward pass whose leaves an eager graph of another stream still holds, whatever the operators in it.)"""
    cases = []
    for t, i in ((5, 304), (300, 88)):
        x, w, dh = _case(t, 1024, i, torch.bfloat16, t)
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        xe, we = xs.detach().requires_grad_(), ws.detach().requires_grad_()
        alive = fso.ffn.gated_linear(xe, we)
        torch.autograd.grad(alive, (xe, we), dh, retain_graph=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h = fso.ffn.gated_linear(xs, ws)
            dx, dw = torch.autograd.grad(h, (xs, ws), dh)
        cases.append((graph, xs, ws, dh, h, dx, dw, alive))
    for seed in (1, 2):
        for graph, xs, ws, dh, *_ in cases:
            with torch.no_grad():
                xs.copy_(R.rows(*xs.shape, seed, xs.dtype))
                dh.copy_(R.rows(*dh.shape, seed + 9, dh.dtype))
        for c in cases:
            c[0].replay()
        for c in reversed(cases):
            c[0].replay()
        torch.cuda.synchronize()
        for _, xs, ws, dh, h, dx, dw, _ in cases:
            for a, b in zip((h.detach(), dx, dw), _grads(fso, xs, ws, dh, "silu")):
                assert torch.equal(a, b)


def test_compiled_with_gradients(fso, device_ok):
    x, w, dh = _case(33, 72, 40, torch.bfloat16)
    f = torch.compile(lambda a, b: fso.ffn.gated_linear(a, b, activation="gelu_tanh"), backend="aot_eager", fullgraph=True)
    want = _grads(fso, x, w, dh, "gelu_tanh")
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    h = f(xr, wr)
    for a, b in zip((h.detach(), *torch.autograd.grad(h, (xr, wr), dh)), want):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(f(x, w), fso.ffn.gated_linear(x, w, activation="gelu_tanh"))


def test_second_derivatives_are_refused(fso, device_ok):
    x, w, _ = _case(4, 16, 8, torch.bfloat16)
    x.requires_grad_()
    (g,) = torch.autograd.grad(fso.ffn.gated_linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_trained_in_16_bits_served_in_4(fso, device_ok):
    """A step of gradient descent on the gated projection, then the same weights in 4 bits: the 4-bit projection is the 16-bit
    one of the dequantized weights, and the chain into a 4-bit down projection is its definition's."""
    t, k, i = 6, 256, 192
    x, w, dh = _case(t, k, i, torch.bfloat16, 3)
    down = R.rows(k, i, 9, torch.bfloat16, std=i ** -0.5).cuda()
    w = w.requires_grad_()
    fso.ffn.gated_linear(x, w).backward(dh)
    with torch.no_grad():
        w -= 0.01 * w.grad
    gate_up = fso.int4.quantize_weight(w, group_size=32, zero_point=True)
    down4 = fso.int4.quantize_weight(down, group_size=64)
    wd = R.dequantize(gate_up.codes, gate_up.scale, gate_up.zero)
    h, bound, _, _ = R.gated(x, wd, "silu")
    got = fso.int4.gated_linear(x, gate_up)
    R.inside(got, h, bound, "4-bit gated projection")
    y = got.double() @ R.dequantize(down4.codes, down4.scale, down4.zero).t()
    mag = got.double().abs() @ R.dequantize(down4.codes, down4.scale, down4.zero).abs().t()
    R.inside(fso.int4.linear(got, down4), y, R.half_step(x.dtype) * y.abs() + R.sum_error(i) * mag, "4-bit down projection")
    # Rounding to 4 bits moves a weight by at most half a step, and one at the end of its group's range, 15 steps wide, by up
    # to 15 times the rounding of the step to bf16 more: a step stored 2^-8 short ends its codes 15 * 2^-8 steps early.
    step = gate_up.scale.double().repeat_interleave(32, 1)
    assert ((wd - w.detach().double()).abs() <= (0.5 + 15 * R.half_step(torch.bfloat16) + 1e-3) * step).all()
