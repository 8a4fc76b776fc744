"""bf16 products grouped by expert and their gradients against 64 bits.

A sum of d products of bf16 in f32, in any order and with each addition cut off instead of rounded, is off by at most
d 2^-23 times the sum of the products' magnitudes; a bf16 output adds 2^-8 of the value, an addition to f32 2^-23 of the result."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import grouped, ops        # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
FORMS = ["forward", "by_input", "by_weight"]


def reference(form, x, dy, w, offsets):
    """The form's result and the sum of magnitudes behind each element, f64; rows of no group NaN."""
    cuts = [min(c, x.shape[0]) for c in offsets]
    if form == "by_weight":
        value = torch.zeros(len(cuts) - 1, dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
    else:
        value = torch.full((x.shape[0], dy.shape[1] if form == "forward" else x.shape[1]), torch.nan, dtype=torch.float64, device=x.device)
    size = value.clone()
    for g in range(len(cuts) - 1):
        begin, end = cuts[g], max(cuts[g], cuts[g + 1])
        if form == "by_weight":
            a, b = dy[begin:end].double().t(), x[begin:end].double()
            value[g], size[g] = a @ b, a.abs() @ b.abs()
        elif end > begin:
            a = (x if form == "forward" else dy)[begin:end].double()
            b = w[g].double().t() if form == "forward" else w[g].double()
            value[begin:end], size[begin:end] = a @ b, a.abs() @ b.abs()
    return value, size


def depth_of(form, n, k, offsets):
    if form == "by_weight":
        return max([1] + [b - a for a, b in zip(offsets, offsets[1:])])
    return k if form == "forward" else n


def run(form, x, dy, w, offsets, **more):
    if form == "by_weight":
        return grouped.GroupedWeightGradient(w.shape[0], w.shape[1], w.shape[2]).forward(dy, x, offsets, **more)
    product = grouped.GroupedProduct(w)
    return product.forward(x, offsets, **more) if form == "forward" else product.by_input(dy, offsets, **more)


def inputs(seed, rows, groups, n, k):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF16)  # noqa: E731
    return normal(rows, k), normal(rows, n), normal(groups, n, k)


def on_device(offsets):
    return torch.tensor(offsets, dtype=torch.int32, device="cuda")


def check(got, value, size, depth, dtype):
    here = ~torch.isnan(value)
    err = (got.double() - value).abs()[here]
    bound = (depth * 2.0 ** -23 * size + (2.0 ** -8 if dtype is BF16 else 2.0 ** -23) * value.abs())[here]
    assert torch.isfinite(got.double()[here]).all()
    assert bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))


# (rows, offsets): sizes around the tiles' borders, empty groups, rows of no group in front and behind
RAGGED = [
    (1, [0, 1]),
    (1, [0, 0, 0, 1, 1]),
    (5, [0, 1, 2, 3, 4, 5]),
    (16, [0, 15, 15, 16]),
    (33, [0, 32, 33]),
    (130, [3, 20, 20, 61, 127]),
    (300, [0, 256, 300]),
    (700, [0, 257, 258, 515, 700]),
    (1100, [0, 0, 1025, 1025, 1100]),
    (64, [0, 0, 0]),
]
SIZES = [(8, 8), (16, 64), (264, 72), (128, 520), (520, 256), (1032, 64), (64, 1544)]
ODD = [(7, 33), (1, 1), (65, 130), (12, 20)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n,k", SIZES + ODD)
@pytest.mark.parametrize("case", range(len(RAGGED)))
def test_against_64_bits(form, n, k, case):
    rows, offsets = RAGGED[case]
    x, dy, w = inputs(case * 100 + n + k, rows, len(offsets) - 1, n, k)
    value, size = reference(form, x, dy, w, offsets)
    for dtype in (BF16, F32):
        got = run(form, x, dy, w, on_device(offsets), dtype=dtype)
        assert got.dtype is dtype and got.shape == value.shape
        check(got, value, size, depth_of(form, n, k, offsets), dtype)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n,k,rows,groups", [(2048, 1024, 1500, 4), (384, 7168, 40, 16), (7168, 256, 300, 3), (512, 512, 9000, 2)])
def test_larger(form, n, k, rows, groups):
    g = torch.Generator().manual_seed(rows)
    offsets = [0] + sorted(torch.randint(0, rows + 1, (groups - 1,), generator=g).tolist()) + [rows]
    x, dy, w = inputs(rows, rows, groups, n, k)
    value, size = reference(form, x, dy, w, offsets)
    for dtype in (BF16, F32):
        check(run(form, x, dy, w, on_device(offsets), dtype=dtype), value, size, depth_of(form, n, k, offsets), dtype)


@pytest.mark.parametrize("form", ["forward", "by_input"])
@pytest.mark.parametrize("rows", [8, 300, 2500])
@pytest.mark.parametrize("depth", [1024, 1025 * 8, 7168])
def test_deep_sums_in_f32(form, rows, depth):
    """An accumulator takes 64 additions of 16 products, each cut off by 2^-23 of the sum at most, then segments are added
    with rounding (at most 9 here): 64 x 2^-23 and 9 x 2^-24 of what has been summed, which is below the result's norm."""
    wide = 520
    x, dy, w = inputs(rows + depth, rows, 1, *((wide, depth) if form == "forward" else (depth, wide)))
    value, _ = reference(form, x, dy, w, [0, rows])
    got = run(form, x, dy, w, on_device([0, rows]), dtype=F32)
    assert float((got.double() - value).norm() / value.norm()) <= 64 * 2.0 ** -23 + 9 * 2.0 ** -24


@pytest.mark.parametrize("n,k,groups,rows", [(520, 264, 1, 3001), (2048, 1032, 6, 9011), (72, 40, 4, 30000)])
def test_deep_gradients_in_f32(n, k, groups, rows):
    """The same of the weight's gradient, whose depth is a group's rows (here equally many)."""
    x, dy, w = inputs(rows, rows, groups, n, k)
    offsets = [rows * i // groups for i in range(groups + 1)]
    value, _ = reference("by_weight", x, dy, w, offsets)
    got = run("by_weight", x, dy, w, on_device(offsets), dtype=F32)
    assert float((got.double() - value).norm() / value.norm()) <= 64 * 2.0 ** -23 + 31 * 2.0 ** -24


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("groups", [1, 1000, 1024])
def test_numbers_of_groups(form, groups):
    rows, n, k = 700, 24, 40
    g = torch.Generator().manual_seed(groups)
    offsets = [0] + sorted(torch.randint(0, rows + 1, (groups - 1,), generator=g).tolist()) + [rows]
    x, dy, w = inputs(groups, rows, groups, n, k)
    value, size = reference(form, x, dy, w, offsets)
    check(run(form, x, dy, w, on_device(offsets), dtype=F32), value, size, depth_of(form, n, k, offsets), F32)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n,k", [(264, 136), (33, 7)])
def test_added_to_what_is_there(form, n, k):
    rows, offsets = 300, [2, 100, 100, 290]
    x, dy, w = inputs(4, rows, 3, n, k)
    value, size = reference(form, x, dy, w, offsets)
    into = torch.randn(value.shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    before = into.clone()
    assert run(form, x, dy, w, on_device(offsets), into=into) is into
    check(into, value + before.double(), size + before.double().abs(), depth_of(form, n, k, offsets) + 1, F32)
    untouched = torch.isnan(value)
    assert torch.equal(into[untouched], before[untouched])
    if form == "by_weight":
        assert torch.equal(into[1], before[1])                             # the group without rows


@pytest.mark.parametrize("form", ["forward", "by_input"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", [(264, 136), (33, 7)])
def test_rows_of_no_group_are_left_as_they_are(form, dtype, n, k):
    rows, offsets = 200, [17, 18, 18, 150]
    x, dy, w = inputs(5, rows, 3, n, k)
    out = torch.full((rows, n if form == "forward" else k), 7.0, dtype=dtype, device="cuda")
    guard = out.clone()
    assert run(form, x, dy, w, on_device(offsets), out=out) is out
    assert torch.equal(out[:17], guard[:17]) and torch.equal(out[150:], guard[150:])
    value, size = reference(form, x, dy, w, offsets)
    check(out, value, size, depth_of(form, n, k, offsets), dtype)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n,k", [(264, 136), (33, 7)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_where_it_is(form, n, k, bad):
    """In rows of no group, in another group's rows next to this one's, and in another group's matrix."""
    rows, offsets = 210, [5, 60, 77, 77, 200]
    x, dy, w = inputs(6, rows, 4, n, k)
    for r in (0, 4, 62, 76, 200, 209):
        x[r] = bad
        dy[r] = bad
    w[1] = bad
    clean = offsets[:]
    value, size = reference(form, x, dy, w, clean)
    got = run(form, x, dy, w, on_device(offsets), dtype=F32)
    if form == "by_weight":
        keep = [0, 2, 3]
        check(got[keep], value[keep], size[keep], depth_of(form, n, k, offsets), F32)
        assert not torch.isfinite(got[1]).any()
    else:
        keep = [r for r in range(5, 200) if not 60 <= r < 77]
        check(got[keep], value[keep], size[keep], depth_of(form, n, k, offsets), F32)
        assert not torch.isfinite(got[60:77]).any()


def test_a_row_that_is_not_finite_spoils_no_other_row():
    for form in ("forward", "by_input"):
        x, dy, w = inputs(7, 40, 1, 136, 72)
        want = run(form, x, dy, w, on_device([0, 40]))
        x[13] = float("nan")
        dy[13] = float("nan")
        got = run(form, x, dy, w, on_device([0, 40]))
        assert torch.isnan(got[13]).all()
        keep = [r for r in range(40) if r != 13]
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n,k", [(264, 136), (33, 7)])
def test_offsets_that_are_no_offsets(form, n, k):
    """Past the rows, descending: every group stays inside the rows."""
    rows = 100
    x, dy, w = inputs(8, rows, 4, n, k)
    for offsets in ([0, 50, 300, 2 ** 31 - 1, 2 ** 31 - 1], [0, 40, 20, 20, 60], [90, 100, 101, 5, 5], [-1, -1, -1, -1, -1]):
        dev = on_device(offsets)
        unsigned = [o & 0xffffffff for o in offsets]
        got = run(form, x, dy, w, dev, dtype=F32)
        torch.cuda.synchronize()
        if form == "by_weight":
            value, size = reference(form, x, dy, w, unsigned)
            check(got, value, size, rows, F32)
    assert ops.k3_moe_device_status() == 0


@pytest.mark.parametrize("form", FORMS)
def test_the_same_call_gives_the_same_bits(form):
    rows, offsets = 1300, [0, 3, 400, 401, 1300]
    x, dy, w = inputs(9, rows, 4, 776, 520)
    dev = on_device(offsets)
    want = run(form, x, dy, w, dev, dtype=F32)
    for _ in range(5):
        assert torch.equal(run(form, x, dy, w, dev, dtype=F32), want)


@pytest.mark.parametrize("form", FORMS)
def test_captured_with_other_offsets_on_replay(form):
    """A graph reads the offsets that the buffer holds when it is replayed."""
    rows, n, k = 400, 264, 136
    x, dy, w = inputs(10, rows, 3, n, k)
    dev = on_device([0, 100, 300, 400])
    product, gradient = grouped.GroupedProduct(w), grouped.GroupedWeightGradient(3, n, k)
    call = {"forward": lambda: product.forward(x, dev, dtype=F32), "by_input": lambda: product.by_input(dy, dev, dtype=F32),
            "by_weight": lambda: gradient.forward(dy, x, dev)}[form]
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    big = inputs(11, 9000, 3, n, k)                                         # the object serves a larger call in between
    more = on_device([0, 1000, 8000, 9000])
    {"forward": lambda: product.forward(big[0], more), "by_input": lambda: product.by_input(big[1], more),
     "by_weight": lambda: gradient.forward(big[1], big[0], more)}[form]()
    for offsets in ([0, 100, 300, 400], [0, 0, 0, 400], [0, 1, 399, 400]):
        dev.copy_(on_device(offsets))
        graph.replay()
        value, size = reference(form, x, dy, w, offsets)
        check(out, value, size, depth_of(form, n, k, offsets), F32)


@pytest.mark.parametrize("form", FORMS)
def test_two_objects_on_two_streams(form):
    """Inputs made on the current stream, calls on two others at once."""
    rows, n, k, offsets = 900, 520, 264, [0, 300, 301, 900]
    dev = on_device(offsets)
    first, second = inputs(12, rows, 3, n, k), inputs(13, rows, 3, n, k)
    want = [run(form, *first, dev, dtype=F32), run(form, *second, dev, dtype=F32)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, data in zip(streams, (first, second)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run(form, *data, dev, dtype=F32))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_rows():
    x, dy, w = inputs(14, 0, 2, 16, 24)
    dev = on_device([0, 0, 0])
    assert run("forward", x, dy, w, dev).shape == (0, 16) and run("by_input", x, dy, w, dev).shape == (0, 24)
    assert not run("by_weight", x, dy, w, dev).any()
    out = torch.ones(2, 16, 24, device="cuda")
    assert torch.equal(run("by_weight", x, dy, w, dev, into=out), torch.ones_like(out))
    assert not run("by_weight", x, dy, w, dev, out=out).any()


def test_rows_that_do_not_start_on_16_bytes():
    """The same values from memory that the TMA unit cannot read."""
    rows, n, k, offsets = 90, 136, 72, [0, 40, 90]
    x, dy, w = inputs(15, rows, 2, n, k)
    odd = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    dev = on_device(offsets)
    for form in FORMS:
        value, size = reference(form, x, dy, w, offsets)
        check(run(form, odd(x), odd(dy), odd(w), dev, dtype=F32), value, size, depth_of(form, n, k, offsets), F32)
        out = torch.zeros(value.numel() + 1, dtype=BF16, device="cuda")[1:].view(value.shape)
        check(run(form, x, dy, w, dev, out=out), value, size, depth_of(form, n, k, offsets), BF16)


def spread(groups, sizes, front=0):
    """Offsets of groups whose sizes go through `sizes` in turn, rows of no group in front."""
    cuts = [front]
    for g in range(groups):
        cuts.append(cuts[-1] + sizes[g % len(sizes)])
    return cuts


# few rows per group on average: groups on both sides of 16 rows, which different kernels take, side by side
MIXED = [[1], [3, 0, 16, 0, 1], [15, 17, 0, 0, 2], [0] * 40 + [130, 16, 0, 1, 33], [0] * 895 + [1200], [16, 0, 0]]


@pytest.mark.parametrize("n,k", [(264, 136), (40, 520), (1032, 64), (72, 264)])
@pytest.mark.parametrize("case", range(len(MIXED)))
def test_gradients_of_small_groups_beside_large_ones(n, k, case):
    offsets = spread(896, MIXED[case], front=3)
    rows = offsets[-1] + 5
    x, dy, w = inputs(case, rows, 896, n, k)
    x[:3], x[-5:], dy[:3], dy[-5:] = float("nan"), float("nan"), float("inf"), float("nan")
    value, size = reference("by_weight", x, dy, w, offsets)
    depth = depth_of("by_weight", n, k, offsets)
    for dtype in (BF16, F32):
        check(run("by_weight", x, dy, w, on_device(offsets), dtype=dtype), value, size, depth, dtype)
    into = torch.randn(value.shape, generator=torch.Generator(device="cuda").manual_seed(case), device="cuda")
    before = into.clone()
    run("by_weight", x, dy, w, on_device(offsets), into=into)
    check(into, value + before.double(), size + before.double().abs(), depth + 1, F32)
    empty = [g for g in range(896) if offsets[g] == offsets[g + 1]]
    assert torch.equal(into[empty], before[empty])


@pytest.mark.parametrize("rows", [1, 7, 16, 60])
@pytest.mark.parametrize("n,k", [(2120, 2056), (72, 15368)])
def test_gradients_of_a_few_rows_of_large_matrices(rows, n, k):
    groups = 12
    offsets = spread(groups, [rows // groups])[:-1] + [rows]
    x, dy, w = inputs(rows, rows, groups, n, k)
    value, size = reference("by_weight", x, dy, w, offsets)
    for dtype in (BF16, F32):
        check(run("by_weight", x, dy, w, on_device(offsets), dtype=dtype), value, size, depth_of("by_weight", n, k, offsets), dtype)


def test_a_row_that_is_not_finite_among_small_groups():
    offsets = spread(896, [2, 16, 17, 1, 0])
    x, dy, w = inputs(16, offsets[-1], 896, 264, 136)
    bad = [5, 6, 7, 401, 895]
    for g in bad:
        if offsets[g] < offsets[g + 1]:
            x[offsets[g]], dy[offsets[g + 1] - 1] = float("nan"), float("inf")
    value, size = reference("by_weight", x, dy, w, offsets)
    got = run("by_weight", x, dy, w, on_device(offsets), dtype=F32)
    keep = [g for g in range(896) if g not in bad]
    check(got[keep], value[keep], size[keep], 17, F32)
    assert not any(bool(torch.isfinite(got[g]).all()) for g in bad if offsets[g] < offsets[g + 1])


def test_captured_with_groups_that_become_large():
    groups, n, k, rows = 896, 264, 136, 4000
    x, dy, w = inputs(17, rows, groups, n, k)
    all_offsets = [spread(groups, s) for s in ([4], [0, 0, 0, 16], [17, 0, 0, 0, 0], [0] * 895 + [4000], [0])]
    dev = on_device(all_offsets[0])
    gradient = grouped.GroupedWeightGradient(groups, n, k)
    gradient.forward(dy, x, dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gradient.forward(dy, x, dev)
    for offsets in all_offsets:
        dev.copy_(on_device(offsets))
        graph.replay()
        value, size = reference("by_weight", x, dy, w, offsets)
        check(out, value, size, depth_of("by_weight", n, k, offsets), F32)
    assert ops.k3_moe_device_status() == 0


@pytest.mark.parametrize("n,k", [(520, 264), (2048, 1032), (264, 520), (384, 2048)])
@pytest.mark.parametrize("sizes", [[3000, 40, 0, 20], [17, 1088, 1089, 1100, 5, 2500], [0, 0, 0, 0, 0, 0, 5000, 1]])
def test_deep_groups_among_others_in_f32(n, k, sizes):
    """An accumulator takes up to 68 additions of 16 products, each cut off by 2^-23 of the sum at most; segments are added
    with rounding, at most 10 here."""
    offsets = spread(len(sizes) * 5, sizes)
    rows = offsets[-1]
    x, dy, w = inputs(n + sizes[0], rows, len(offsets) - 1, n, k)
    value, _ = reference("by_weight", x, dy, w, offsets)
    into = torch.ones(value.shape, device="cuda")
    got = run("by_weight", x, dy, w, on_device(offsets), dtype=F32)
    run("by_weight", x, dy, w, on_device(offsets), into=into)
    for g, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if a == b:
            assert not got[g].any() and bool((into[g] == 1).all())
            continue
        norm = value[g].norm()
        assert float((got[g].double() - value[g]).norm() / norm) <= 68 * 2.0 ** -23 + 10 * 2.0 ** -24
        assert float((into[g].double() - 1 - value[g]).norm()) <= (69 * 2.0 ** -23 + 10 * 2.0 ** -24) * float((value[g].abs() + 1).norm())
    assert ops.k3_moe_device_status() == 0
