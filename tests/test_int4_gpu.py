"""``fso.int4`` against the definition in 64 bits: every element within one rounding of the result plus what fp32 sums of K
terms allow (ffn_reference.sum_error), at row counts, widths and group sizes off every tile."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu

SIZES = [(1, 32, 1, 32), (1, 128, 7, 64), (1, 4096, 100, 128), (2, 96, 65, 32), (3, 2560, 64, 128), (7, 1024, 33, 256),
         (8, 512, 130, 32), (9, 320, 257, 64), (16, 640, 48, 128), (17, 1056, 96, 32), (31, 2048, 40, 2048),
         (33, 192, 300, 64), (64, 768, 129, 128), (65, 512, 70, 128), (200, 384, 140, 64), (1, 14336, 16, 128)]
# more tiles than SMs (whole tiles beside split ones), and than two for each; contractions off the 256-wide steps
MANY = [(2, 1056, 10000, 32), (20, 1120, 19999, 32), (1, 320, 40010, 64), (50, 1152, 38100, 128)]


def _linear_bound(x, w, bias=None):
    y = x.double() @ w.t()
    mag = x.double().abs() @ w.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    he = R.half_step(x.dtype)
    return y, he * y.abs() + R.sum_error(x.shape[1] + 2) * mag + torch.finfo(x.dtype).smallest_normal * he


def _weight(fso, n, k, group, seed, zero, scale_dtype):
    parts = [p if p is None else p.cuda() for p in R.random_int4(n, k, group, seed, zero, scale_dtype)]
    return fso.int4.prepare_weight(*parts), R.dequantize(*parts)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("t,k,n,group", SIZES + MANY)
def test_linear(fso, device_ok, t, k, n, group, dtype):
    scale_dtype = (torch.bfloat16, torch.float16, torch.float32)[(t + n) % 3]
    weight, w = _weight(fso, n, k, group, 10 * t + n, n % 2 == 0, scale_dtype)
    x = R.rows(t, k, t, dtype).cuda()
    y = fso.int4.linear(x, weight)
    assert y.shape == (t, n) and y.dtype == dtype
    R.inside(y, *_linear_bound(x, w))
    bias = R.rows(1, n, 5, dtype)[0].cuda()
    R.inside(fso.int4.linear(x, weight, bias=bias), *_linear_bound(x, w, bias))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("t,k,n,group", SIZES)
def test_gated_linear(fso, device_ok, t, k, n, group, dtype):
    act = R.ACTIVATIONS[(t + n) % 3]
    weight, w = _weight(fso, 2 * n, k, group, t + n, n % 2 == 1, torch.float32)
    x = (R.rows(t, k, t, dtype) / (0.02 * 5 * k ** 0.5)).to(dtype).cuda()
    h, bound, _, _ = R.gated(x, w, act)
    got = fso.int4.gated_linear(x, weight, activation=act)
    assert got.shape == (t, n) and got.dtype == dtype
    R.inside(got, h, bound, act)


def test_every_code_and_zero_point_is_exact(fso, device_ok):
    """One x of 1 in each group: the result is scale * (code - zero), exactly, for all 16 x 16 pairs."""
    k, group = 512, 32
    codes = torch.arange(16, dtype=torch.uint8).repeat(16)                      # row r: code r % 16, zero point r / 16
    zero = torch.arange(16, dtype=torch.uint8).repeat_interleave(16)
    packed = (codes | codes << 4)[:, None].expand(256, k // 2).contiguous().cuda()
    scale = torch.full((256, k // group), 0.5, dtype=torch.bfloat16, device="cuda")
    weight = fso.int4.prepare_weight(packed, scale, zero[:, None].expand(256, k // group).contiguous().cuda())
    want = 0.5 * (codes.float() - zero.float())
    for dtype in R.DTYPES:
        x = torch.zeros(k, k, dtype=dtype, device="cuda").fill_diagonal_(1)     # row t picks out k = t
        for t0, rows in ((0, 1), (37, 8), (64, 64), (0, 512)):
            y = fso.int4.linear(x[t0:t0 + rows], weight)
            assert torch.equal(y.float().cpu(), want.expand(rows, 256))


def test_order_of_the_codes(fso, device_ok):
    """Distinct weights along K, one nonzero x each: every position of the row meets its own x."""
    k = 1024
    codes, scale, _ = R.random_int4(40, k, 64, 3, False, torch.float32)
    weight = fso.int4.prepare_weight(codes.cuda(), scale.cuda())
    x = torch.eye(k, dtype=torch.float16, device="cuda")
    want = R.dequantize(codes, scale, None).t().float().half()
    for lo, hi in ((0, 16), (500, 564), (0, k)):
        assert torch.equal(fso.int4.linear(x[lo:hi], weight).cpu(), want[lo:hi])


def test_rows_are_read_where_they_lie(fso, device_ok):
    k, n, t = 256, 96, 12
    weight, _ = _weight(fso, n, k, 64, 1, True, torch.bfloat16)
    buf = R.rows(2 * t, k + 40, 1, torch.bfloat16).cuda()
    for name, x in {"slice": buf[:t, 8:8 + k], "off the boundary": buf[:t, 3:3 + k], "every second row": buf[::2, :k],
                    "expanded": buf[5:6, :k].expand(t, k), "columns apart": buf[:t].t().contiguous().t()[:, :k],
                    "three dimensions": buf[:, :k].view(2, t, k), "one row": buf[3, :k]}.items():
        y, h = fso.int4.linear(x, weight), fso.int4.gated_linear(x, weight)
        assert y.shape == x.shape[:-1] + (n,) and h.shape == x.shape[:-1] + (n // 2,), name
        assert torch.equal(y, fso.int4.linear(x.contiguous(), weight)), name
        assert torch.equal(h, fso.int4.gated_linear(x.contiguous(), weight)), name
    assert fso.int4.linear(buf[:0, :k], weight).shape == (0, n)
    assert fso.int4.gated_linear(torch.empty(2, 0, k, dtype=torch.float16, device="cuda"), weight).shape == (2, 0, n // 2)


def test_extreme_values_stay_in_their_row(fso, device_ok):
    k, n = 512, 40
    weight, w = _weight(fso, n, k, 128, 2, True, torch.bfloat16)
    x = R.rows(20, k, 1, torch.bfloat16).cuda()
    want = fso.int4.linear(x, weight)
    y = x.clone()
    y[3, 5] = float("nan")
    y[11, 200] = float("inf")
    y[12] = 0
    got = fso.int4.linear(y, weight)
    keep = torch.ones(20, dtype=torch.bool, device="cuda")
    keep[[3, 11, 12]] = False
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[3]).all() and not got[12].any()
    # an infinity times a weight of sign s is an infinity of that sign, times a weight of zero not a number
    inf = torch.where(w[:, 200] == 0, torch.nan, torch.sign(w[:, 200]) * torch.inf).to(torch.bfloat16)
    assert torch.equal(torch.nan_to_num(got[11], nan=7.0), torch.nan_to_num(inf, nan=7.0))


@pytest.mark.parametrize("power", [-126, -116, 100, 116])
def test_rows_of_any_magnitude(fso, device_ok, power):
    """bf16 rows around the smallest normal numbers and near the largest: the same bound as everywhere."""
    weight, w = _weight(fso, 64, 256, 64, 3, True, torch.float32)
    x = (R.rows(4, 256, 1, torch.float32) * 2.0 ** power).to(torch.bfloat16).cuda()
    R.inside(fso.int4.linear(x, weight), *_linear_bound(x, w))


def test_quantized_weights_are_the_nearest_steps(fso, device_ok):
    for dtype in R.DTYPES:
        for group in fso.int4.GROUP_SIZES:
            w = R.rows(37, 1536 // group * group, group, dtype, std=0.02)
            w[3, :group] = 0
            w[4, :group] = w[4, :group].abs()
            for zero_point in (False, True):
                q = fso.int4.quantize_weight(w.cuda(), group_size=group, zero_point=zero_point, scale_dtype=torch.float32)
                assert q.group_size == group and (q.zero is None) == (not zero_point)
                d = R.dequantize(q.codes.cpu(), q.scale.cpu(), None if q.zero is None else q.zero.cpu())
                v = w.double().view(37, -1, group)
                span = v.amax(-1).clamp(min=0) - v.amin(-1).clamp(max=0)
                step = span / 15 if zero_point else v.abs().amax(-1) / 7
                assert torch.allclose(q.scale.cpu().double(), step, rtol=1e-6, atol=0)
                # half a step, and fp32 quotients that are off by a few units next to a border
                assert ((d.view_as(v) - v).abs() <= 0.5 * step[..., None] * (1 + 1e-4)).all()
                assert not d[3, :group].any()


def test_quantizing_does_not_hide_a_nan(fso, device_ok):
    for group in fso.int4.GROUP_SIZES:
        w = R.rows(5, 512, group, torch.bfloat16, std=0.02)
        w[1, 300] = float("nan")
        w[3, 511] = float("-inf")
        for zero_point in (False, True):
            q = fso.int4.quantize_weight(w.cuda(), group_size=group, zero_point=zero_point)
            want = torch.zeros(5, 512 // group, dtype=torch.bool)
            want[1, 300 // group] = want[3, 511 // group] = True
            assert torch.equal(torch.isnan(q.scale.cpu()), want)
            y = fso.int4.linear(torch.ones(2, 512, dtype=torch.bfloat16, device="cuda"), q).cpu()
            assert torch.equal(torch.isnan(y), torch.tensor([False, True, False, True, False]).expand(2, 5))


def test_same_bits_every_time_and_on_another_stream(fso, device_ok):
    weight, _ = _weight(fso, 640, 2048, 64, 2, True, torch.bfloat16)
    side = torch.cuda.Stream()
    for t in (1, 16, 40):
        x = R.rows(t, 2048, t, torch.bfloat16).cuda()
        first = fso.int4.linear(x, weight), fso.int4.gated_linear(x, weight)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = fso.int4.linear(x, weight), fso.int4.gated_linear(x, weight)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, other))
        assert torch.equal(first[0], fso.int4.linear(x, weight))


def test_a_handle_has_memory_of_its_own(fso, device_ok):
    """What the caller does to its tensors afterwards does not reach the handle, whatever their shapes."""
    for n, groups in ((32, 1), (64, 3), (33, 1), (1, 4)):
        codes, scale, zero = (p.cuda() for p in R.random_int4(n, 32 * groups, 32, n))
        weight = fso.int4.prepare_weight(codes, scale, zero)
        kept = [t.clone() for t in (codes, scale, zero)]
        for t in (codes, scale, zero):
            t.zero_()
        for got, want in zip((weight.codes, weight.scale, weight.zero), kept):
            assert torch.equal(got, want)
        x = R.rows(2, 32 * groups, 1, torch.bfloat16).cuda()
        R.inside(fso.int4.linear(x, weight), *_linear_bound(x, R.dequantize(*kept)))


def test_captured_decode_steps(fso, device_ok):
    """Two captured feed-forwards (gated projection, down projection) of different sizes, replayed in turn on new inputs."""
    graphs = []
    for t, k, i in ((1, 1024, 512), (20, 512, 288)):
        gate_up, _ = _weight(fso, 2 * i, k, 32, t, True, torch.bfloat16)
        down, _ = _weight(fso, k, i, 32, t + 1, False, torch.bfloat16)
        x = R.rows(t, k, t, torch.bfloat16).cuda()
        step = lambda x=x, a=gate_up, b=down: fso.int4.linear(fso.int4.gated_linear(x, a), b)  # noqa: E731
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step()
        graphs.append((g, x, y, step))
    for seed in range(3):
        for g, x, _, _ in graphs:
            x.copy_(R.rows(*x.shape, seed, x.dtype))
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, _, y, step in graphs:
            assert torch.equal(y, step())


def test_compiled(fso, device_ok):
    weight, _ = _weight(fso, 64, 128, 32, 2, True, torch.bfloat16)
    x = R.rows(3, 128, 1, torch.bfloat16).cuda()
    f = torch.compile(lambda a: (fso.int4.linear(a, weight), fso.int4.gated_linear(a, weight)), backend="aot_eager",
                      fullgraph=True)
    y, h = f(x)
    assert torch.equal(y, fso.int4.linear(x, weight)) and torch.equal(h, fso.int4.gated_linear(x, weight))
