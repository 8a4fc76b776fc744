"""RMS norm with the residual's addition and E4M3 codes, and its gradient, against 64 bits.

A row's sum runs through at most 64 products per thread and a tree of 10, in f32: 80 roundings of 2^-24, of a sum of squares
half of that in rstd.  A bf16 output adds 2^-8 of the value, a code 2^-4 of it or half of the smallest step, 2^-10 scales."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import fp8, norm, ops        # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
EPSILON = 1e-5
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
SUM = 80 * 2.0 ** -24
# row lengths around the changes of kernel (1024, 2048, 4096, 8192) and of a block of 128, whole vectors and not
HIDDEN = [1, 7, 8, 16, 127, 128, 129, 136, 256, 257, 512, 1000, 1024, 1025, 1032, 2048, 2056, 3583, 4096, 4104, 7168, 8192, 8200, 16384]


def inputs(seed, rows, hidden, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda d: (torch.randn(rows, hidden, generator=g, device="cuda") * scale).to(d)  # noqa: E731
    weight = (1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(BF16)
    return normal(dtype), normal(dtype), normal(BF16), normal(dtype), weight


def check(got, want, bound):
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))


def check_forward(r, x, residual, weight):
    rows, hidden = x.shape
    if residual is None:
        assert r.sum is x
    else:
        want = x.double() + residual.double()
        check(r.sum, want, HALF[x.dtype] * want.abs())
    h = r.sum.double()
    rstd = 1 / torch.sqrt(h.square().mean(1) + EPSILON)
    check(r.rstd, rstd, SUM * rstd)
    y = h * rstd.unsqueeze(1) * weight.double()
    if r.y is not None:
        assert r.y.dtype is BF16
        check(r.y, y, (HALF[BF16] + 2 * SUM) * y.abs())
    if r.codes is not None:
        blocks = fp8.blocks(hidden)
        assert r.codes.shape == (rows, fp8.pitch(hidden)) and r.scales.shape == (rows, fp8.scale_pitch(hidden))
        assert not r.codes.view(torch.uint8)[:, hidden:].any() and not r.scales[:, blocks:].any()
        largest = torch.nn.functional.pad(y.abs(), (0, blocks * 128 - hidden)).view(rows, blocks, 128).amax(2)
        scale = (largest / 448).clamp(min=2.0 ** -126)
        check(r.scales[:, :blocks], scale, 2 * SUM * scale)
        full = r.scales[:, :blocks].double().repeat_interleave(128, 1)[:, :hidden]
        check(r.codes[:, :hidden].double() * full, y, (2.0 ** -4 + 4 * SUM) * y.abs() + 2.0 ** -10 * full)


@pytest.mark.parametrize("hidden", HIDDEN)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 9, 700])
def test_forward(hidden, dtype, rows):
    x, residual, _, _, weight = inputs(hidden + rows, rows, hidden, dtype)
    call = norm.RmsNorm(weight, EPSILON)
    for res, y, codes in ((None, True, False), (residual, False, True), (residual, True, True)):
        check_forward(call.forward(x, res, y=y, codes=codes), x, res, weight)
    assert ops.k3_moe_device_status() == 0


def gradient(dy, s, rstd, d_sum, weight):
    """dx and d_weight by the formula in 64 bits, and the magnitudes of what is added up to them."""
    h, g = s.double() * rstd.double().unsqueeze(1), dy.double() * weight.double()
    r = rstd.double().unsqueeze(1)
    dx = r * (g - h * (g * h).mean(1, keepdim=True))
    size = r * (g.abs() + h.abs() * (g * h).abs().mean(1, keepdim=True))
    if d_sum is not None:
        dx, size = dx + d_sum.double(), size + d_sum.double().abs()
    return dx, size, (dy.double() * h).sum(0), (dy.double() * h).abs().sum(0)


@pytest.mark.parametrize("hidden", HIDDEN)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 9, 700])
def test_backward(hidden, dtype, rows):
    s, _, dy, d_sum, weight = inputs(hidden * 3 + rows, rows, hidden, dtype)
    call = norm.RmsNorm(weight, EPSILON)
    rstd = torch.rsqrt(s.double().square().mean(1) + EPSILON).float()
    for extra in (None, d_sum):
        want, size, want_w, size_w = gradient(dy, s, rstd, extra, weight)
        dx, d_weight = call.backward(dy, s, rstd, extra)
        assert dx.dtype is dtype and d_weight.dtype is F32
        check(dx, want, HALF[dtype] * want.abs() + 2 * SUM * size)
        check(d_weight, want_w, (rows + 4) * 2.0 ** -24 * size_w)
        into = torch.ones_like(d_weight)
        _, again = call.backward(dy, s, rstd, extra, into=into)
        assert again is into
        check(into, want_w + 1, (rows + 5) * 2.0 ** -24 * (size_w + 1))
    assert ops.k3_moe_device_status() == 0


def test_gradient_against_differences():
    """The sum of dy y + d_sum s along a direction, in 64 bits, against the kernel's gradients."""
    rows, hidden = 6, 520
    x, residual, dy, d_sum, weight = inputs(5, rows, hidden, F32)
    call = norm.RmsNorm(weight, EPSILON)
    r = call.forward(x, residual)
    dx, d_weight = call.backward(dy, r.sum, r.rstd, d_sum)

    def value(s, w):
        return (dy.double() * s * torch.rsqrt(s.square().mean(1, keepdim=True) + EPSILON) * w + d_sum.double() * s).sum()
    g = torch.Generator(device="cuda").manual_seed(6)
    for _ in range(4):
        v = torch.randn(rows, hidden, generator=g, device="cuda", dtype=torch.float64)
        u = torch.randn(hidden, generator=g, device="cuda", dtype=torch.float64)
        s, w, step = r.sum.double(), weight.double(), 1e-4
        by_s = (value(s + step * v, w) - value(s - step * v, w)) / (2 * step)
        by_w = (value(s, w + step * u) - value(s, w - step * u)) / (2 * step)
        size_s, size_w = (dx.double() * v).abs().sum(), (d_weight.double() * u).abs().sum()
        # the differences' own error: step^2 / 6 of a third derivative of order one per element
        assert abs(float((dx.double() * v).sum() - by_s)) <= float(2 * SUM * size_s) + 1e-8 * rows * hidden * 50
        assert abs(float((d_weight.double() * u).sum() - by_w)) <= float(2 * SUM * size_w) + 1e-8 * hidden


@pytest.mark.parametrize("rows,hidden", [(700, 7168), (5, 7168), (40, 200)])
def test_values_that_are_large_small_and_not_finite(rows, hidden):
    x, _, _, _, weight = inputs(7, rows, hidden, F32)
    x[0] = 0.0                                                     # rstd 1 / sqrt(epsilon), results 0
    x[1] *= 1e-18
    x[2] *= 1e15
    x[3, hidden // 2] = float("nan")
    x[4, 5] = float("inf")
    call = norm.RmsNorm(weight, EPSILON)
    r = call.forward(x, y=True, codes=True)
    keep = [i for i in range(rows) if i not in (3, 4)]
    part = norm.Normed(r.sum[keep], r.y[keep], r.codes[keep], r.scales[keep], r.rstd[keep])
    check_forward(norm.Normed(x[keep], *part[1:])._replace(sum=(kept := x[keep])), kept, None, weight)
    assert torch.isnan(r.y[3]).all() and torch.isnan(r.scales[3, :fp8.blocks(hidden)]).all()
    assert float(r.rstd[4]) == 0.0 and torch.isnan(r.y[4, 5]) and torch.isnan(r.scales[4, 0])
    assert not r.codes.view(torch.uint8)[:, hidden:].any() and not r.scales[:, fp8.blocks(hidden):].any()


@pytest.mark.parametrize("rows", [3, 700])
def test_a_row_does_not_depend_on_the_others(rows):
    """Within the kernels of few and of many rows each."""
    x, residual, _, _, weight = inputs(8, rows, 4096, BF16)
    call = norm.RmsNorm(weight, EPSILON)
    want = call.forward(x, residual, codes=True)
    order = torch.randperm(rows, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    got = call.forward(x[order].contiguous(), residual[order].contiguous(), codes=True)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8) if a.dtype is torch.float8_e4m3fn else a, (b.view(torch.uint8) if b.dtype is torch.float8_e4m3fn else b)[order])


@pytest.mark.parametrize("rows,hidden", [(700, 2048), (3, 2048), (700, 96), (700, 2049)])
def test_the_sum_in_place_of_x_or_the_residual(rows, hidden):
    x, residual, _, _, weight = inputs(9, rows, hidden, BF16)
    want = norm.RmsNorm(weight, EPSILON).forward(x, residual)
    for which in range(2):
        a, b = x.clone(), residual.clone()
        y, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
        assert ops.k3_moe_norm((a, b)[which], y, None, None, rstd, a, b, weight, rows, hidden, ops.NORM_BF16, EPSILON)
        assert torch.equal((a, b)[which], want.sum) and torch.equal(y, want.y) and torch.equal(rstd, want.rstd)
    d = torch.randn(rows, hidden, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(BF16)
    call = norm.RmsNorm(weight, EPSILON)
    dx, _ = call.backward(x, want.sum, want.rstd, d)
    assert ops.k3_moe_norm_backward(d, None, x, want.sum, want.rstd, d, weight, rows, hidden, ops.NORM_BF16, 0, None, 0)
    assert torch.equal(d, dx)


def test_no_rows():
    _, _, _, _, weight = inputs(10, 1, 64, BF16)
    call = norm.RmsNorm(weight, EPSILON)
    x = torch.empty(0, 64, dtype=BF16, device="cuda")
    r = call.forward(x, x, codes=True)
    assert r.sum.shape == r.y.shape == (0, 64) and r.codes.shape == (0, 64) and r.rstd.shape == (0,)
    dx, d_weight = call.backward(x, x, r.rstd)
    assert dx.shape == (0, 64) and not d_weight.any()
    into = torch.ones(64, device="cuda")
    assert ops.k3_moe_norm_backward(None, into, None, None, None, None, None, 0, 64, ops.NORM_BF16, 1, None, 0) and bool((into == 1).all())
    assert ops.k3_moe_norm_backward(None, into, None, None, None, None, None, 0, 64, ops.NORM_BF16, 0, None, 0) and not into.any()


@pytest.mark.parametrize("rows", [5, 700])
def test_captured_and_replayed(rows):
    x, residual, dy, d_sum, weight = inputs(11, rows, 2048, BF16)
    call = norm.RmsNorm(weight, EPSILON)

    def both():
        r = call.forward(x, residual, codes=True)
        return (*r, *call.backward(dy, r.sum, r.rstd, d_sum))
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    more = inputs(12, 2000, 2048, BF16)
    call.backward(more[2], more[0], torch.ones(2000, device="cuda"), more[3])   # a larger workspace
    fresh = inputs(13, rows, 2048, BF16)
    for old, new in zip((x, residual, dy, d_sum), fresh):
        old.copy_(new)
    graph.replay()
    for a, b in zip(out, both()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_into_the_linear_layer():
    """Codes of the norm through an 8-bit product: the values that they stand for times those of the table."""
    rows, hidden, wide = 37, 1040, 264
    x, residual, _, _, weight = inputs(14, rows, hidden, BF16)
    table = torch.randn(wide, hidden, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * 0.05
    codes, scales = fp8.quantize_blocks(table)
    linear = fp8.Fp8Linear(codes, scales, wide, hidden)
    r = norm.RmsNorm(weight, EPSILON).forward(x, residual, y=False, codes=True)
    got = linear.forward_codes(r.codes, r.scales)
    left = r.codes[:, :hidden].double() * r.scales.double().repeat_interleave(128, 1)[:, :hidden]
    right = codes[:, :hidden].double() * scales.double().repeat_interleave(128, 0)[:wide].repeat_interleave(128, 1)[:, :hidden]
    want, size = left @ right.t(), left.abs() @ right.abs().t()
    check(got, want, HALF[BF16] * want.abs() + hidden * 2.0 ** -23 * size)
    with pytest.raises(ValueError, match="different numbers of tokens"):
        linear.forward_codes(r.codes, r.scales[:-1])
    with pytest.raises(ValueError, match="codes: expected"):
        linear.forward_codes(r.codes[:, :-16], r.scales)
    assert linear.forward_codes(r.codes[:0], r.scales[:0]).shape == (0, wide)


# no multiple of 8: a row starts anywhere in a vector; around the changes of kernel, whose places are for 7 elements more
ODD = [2, 3, 5, 12, 100, 249, 250, 505, 506, 777, 1017, 1018, 1020, 1023, 2041, 2042, 4089, 4090, 5003, 8185, 8186, 16377, 16378, 16383]


@pytest.mark.parametrize("hidden", ODD)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [2, 37, 301, 1301])
def test_lengths_that_are_no_whole_vectors(hidden, dtype, rows):
    x, residual, dy, d_sum, weight = inputs(hidden + rows, rows, hidden, dtype)
    call = norm.RmsNorm(weight, EPSILON)
    for y, codes in ((True, False), (False, True), (True, True)):
        r = call.forward(x, residual, y=y, codes=codes)
        check_forward(r, x, residual, weight)
    want, size, want_w, size_w = gradient(dy, r.sum, r.rstd, d_sum, weight)
    dx, d_weight = call.backward(dy, r.sum, r.rstd, d_sum)
    check(dx, want, HALF[dtype] * want.abs() + 2 * SUM * size)
    check(d_weight, want_w, (rows + 4) * 2.0 ** -24 * size_w)
    assert ops.k3_moe_device_status() == 0


@pytest.mark.parametrize("hidden", [24, 777, 1024, 3583, 9000])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [3, 700])
def test_rows_that_do_not_start_on_16_bytes(hidden, dtype, rows):
    """Each tensor one element behind such a place; what is in front and behind stays."""
    odd = lambda t: torch.cat([t.new_full((1,), 7.0), t.reshape(-1), t.new_full((1,), 7.0)])[1:-1].view(t.shape)  # noqa: E731
    plain = inputs(hidden - rows, rows, hidden, dtype)
    x, residual, dy, d_sum, weight = map(odd, plain)
    call = norm.RmsNorm(weight, EPSILON)
    r = call.forward(x, residual, codes=True)
    check_forward(r, x, residual, weight)
    want, size, want_w, size_w = gradient(dy, r.sum, r.rstd, d_sum, weight)
    dx, d_weight = call.backward(dy, r.sum, r.rstd, d_sum)
    check(dx, want, HALF[dtype] * want.abs() + 2 * SUM * size)
    check(d_weight, want_w, (rows + 4) * 2.0 ** -24 * size_w)
    guard = torch.full((rows * hidden + 2,), 5.0, dtype=dtype, device="cuda")
    y = torch.full((rows * hidden + 2,), 5.0, dtype=BF16, device="cuda")
    kind = ops.NORM_F32 if dtype is F32 else ops.NORM_BF16
    rstd = torch.empty(rows, device="cuda")
    assert ops.k3_moe_norm(guard[1:], y[1:], None, None, rstd, x, residual, weight, rows, hidden, kind, EPSILON)
    assert torch.equal(guard[1:-1].view(rows, hidden), r.sum)
    assert all(float(t[i]) == 5.0 for t in (guard, y) for i in (0, -1))


@pytest.mark.parametrize("hidden", [3, 250, 777, 2042, 5003])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nothing_behind_the_last_row_is_written_or_read(hidden, dtype):
    """Outputs and inputs as the first part of larger tensors, whose rest is NaN and stays."""
    rows = 13
    longer = lambda t: torch.cat([t.reshape(-1), t.new_full((40,), float("nan"))])  # noqa: E731
    plain = inputs(hidden, rows, hidden, dtype)
    x, residual, dy, d_sum, weight = map(longer, plain)
    kind = ops.NORM_F32 if dtype is F32 else ops.NORM_BF16
    want = norm.RmsNorm(plain[4], EPSILON).forward(plain[0], plain[1])
    out, y, rstd = longer(torch.empty_like(plain[0])), longer(torch.empty_like(plain[2])), torch.empty(rows, device="cuda")
    n = rows * hidden
    assert ops.k3_moe_norm(out, y, None, None, rstd, x, residual, weight, rows, hidden, kind, EPSILON)
    assert torch.equal(out[:n].view(rows, hidden), want.sum) and torch.equal(y[:n].view(rows, hidden), want.y) and torch.equal(rstd, want.rstd)
    dx, _ = norm.RmsNorm(plain[4], EPSILON).backward(plain[2], want.sum, want.rstd, plain[3])
    s, grad = longer(want.sum), longer(torch.empty_like(plain[0]))
    assert ops.k3_moe_norm_backward(grad, None, dy, s, rstd, d_sum, weight, rows, hidden, kind, 0, None, 0)
    assert torch.equal(grad[:n].view(rows, hidden), dx)
    assert all(bool(torch.isnan(t[n:]).all()) for t in (out, y, grad))


@pytest.mark.parametrize("hidden", [1032, 2048, 4096, 4104, 8192])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_about_a_row_or_two_per_sm(hidden, dtype):
    """Where the gradient changes from blocks of a row to rows through a ring, and from one row at a time to two."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for rows in (sms - 1, sms, sms + 1, 2 * sms - 1, 2 * sms, 2 * sms + 1, 3 * sms):
        s, _, dy, d_sum, weight = inputs(hidden + rows, rows, hidden, dtype)
        rstd = torch.rsqrt(s.double().square().mean(1) + EPSILON).float()
        for extra in (None, d_sum):
            want, size, want_w, size_w = gradient(dy, s, rstd, extra, weight)
            dx, d_weight = norm.RmsNorm(weight, EPSILON).backward(dy, s, rstd, extra)
            check(dx, want, HALF[dtype] * want.abs() + 2 * SUM * size)
            check(d_weight, want_w, (rows + 4) * 2.0 ** -24 * size_w)
    assert ops.k3_moe_device_status() == 0
