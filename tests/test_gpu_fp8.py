"""E4M3 block-scaled operators against plain statements of them: quantisers and layouts bit for bit, products
within the rounding of their sums, experts within that of their stored intermediates."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import fp8, ops            # noqa: E402
from tests import fp8_reference as R           # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
E4M3 = torch.float8_e4m3fn


def normal(seed, *shape, scale=1.0, dtype=BF16):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale
    return x.to(dtype)


def raw(t):
    return t.cpu().contiguous().view(torch.uint8)


def same_codes(got, want):
    """Equal codes; NaN has two."""
    g, w = raw(got), raw(want)
    return bool((((g == w) | ((g & 127 == 127) & (w & 127 == 127)))).all())


def same_scales(got, want):
    return torch.equal(torch.nan_to_num(got.cpu(), nan=-1.0), torch.nan_to_num(want, nan=-1.0))


def check_quantized(form, x, codes, scales):
    rows, columns = x.shape
    src = x.cpu().t().contiguous() if form == "columns" else x.cpu()
    want, want_scales = R.quantize(src, R.BLOCK if form == "blocks" else 1)
    inner = src.shape[1]
    assert same_codes(codes[:, :inner], want)
    assert not raw(codes[:, inner:]).any()                                  # padding is zeros
    n = want_scales.shape[1]
    assert same_scales(scales[:, :n], want_scales)
    if form != "blocks":
        assert not scales[:, n:].cpu().any()


SIZES = [(1, 1), (1, 7168), (3, 127), (5, 128), (129, 129), (16, 1000), (127, 520), (257, 2056), (300, 40), (1000, 33)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("form", ["rows", "columns", "blocks"])
@pytest.mark.parametrize("rows,columns", SIZES)
def test_quantisers(form, rows, columns, dtype):
    x = normal(rows * 7 + columns, rows, columns, dtype=dtype)
    x[:, ::5] *= 30
    x = x.cuda()
    check_quantized(form, x, *getattr(fp8, "quantize_" + form)(x))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("form", ["rows", "columns", "blocks"])
def test_quantisers_at_the_edges_of_the_values(form, dtype):
    x = normal(1, 260, 260, dtype=dtype)
    x[0:128, 0:128] = 0                                                     # a block of zeros
    x[0, 130] = float("inf")
    x[140, 5] = float("nan")
    x[200:, 200:] *= 1e-38 / 4                                              # small and subnormal
    x[130:132, 130:132] = torch.finfo(dtype).max
    x[256:, :] = -0.0
    x = x.cuda()
    check_quantized(form, x, *getattr(fp8, "quantize_" + form)(x))


@pytest.mark.parametrize("form", ["rows", "columns", "blocks"])
def test_quantisers_where_quotients_fall_between_two_codes(form):
    # the largest magnitude is 448 / 2^9, so x * 2^9 is the quotient: every bf16 value of a binade, ties included
    x = (torch.arange(128 * 128).reshape(128, 128) % 448).float() / 16
    x[:, 0], x[0, :] = 28, 28
    x = (x / 512).to(BF16).cuda()
    check_quantized(form, x, *getattr(fp8, "quantize_" + form)(x))


def test_quotients_by_every_kind_of_scale():
    """Scales of all exponents with mantissas at both ends (all ones: the reciprocal that Newton's iteration misses) and
    in between, and quotients at and beside the middle of two codes."""
    bits = torch.arange(2, 245, dtype=torch.int32).repeat_interleave(16) << 23
    g = torch.Generator().manual_seed(4)
    ends = torch.tensor([0x7fffff, 0x7ffffe, 0x7ffffd, 0, 1, 2], dtype=torch.int32)
    mantissas = torch.cat([ends, torch.randint(0, 1 << 23, (10,), generator=g, dtype=torch.int32)]).repeat(bits.numel() // 16)
    scales = (bits | mantissas).view(F32)
    middles = torch.tensor([(8 + m + 0.5) * 2.0 ** (e - 10) for e in range(16) for m in range(8)])[:126]
    x = scales[:, None] * torch.cat([torch.tensor([448.0]), middles, torch.tensor([0.0])])[None]
    x[:, 1:127:3] = torch.nextafter(x[:, 1:127:3], torch.tensor(0.0))
    x[:, 2:127:3] = torch.nextafter(x[:, 2:127:3], torch.tensor(float("inf")))
    x[:, 1:127:2] *= -1
    assert ((x[:, 0] / 448).view(torch.int32) & 0x7fffff == 0x7fffff).sum() > 200
    x = x.cuda()
    check_quantized("rows", x, *fp8.quantize_rows(x))


@pytest.mark.parametrize("form", ["rows", "columns", "blocks"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantisers_take_any_start(form, dtype):
    """A matrix that starts between 16-byte boundaries."""
    rows, columns = 70, 264
    store = normal(9, rows * columns + 1, dtype=dtype).cuda()
    x = store[1:].view(rows, columns)
    check_quantized(form, x, *getattr(fp8, "quantize_" + form)(x))


@pytest.mark.parametrize("rows,columns", [(1, 1), (130, 300), (128, 256), (17, 1000)])
def test_transposed_table(rows, columns):
    codes, scales = fp8.quantize_blocks(normal(3, rows, columns).cuda())
    t, ts = fp8.transpose_blocks(codes, scales, rows, columns)
    assert torch.equal(raw(t[:, :rows]), raw(codes[:, :columns]).t())
    assert not raw(t[:, rows:]).any()
    assert torch.equal(ts.cpu(), scales.cpu().t())


def dirty(codes, width):
    """Padding bytes that are NaN codes: none may enter a sum."""
    codes.view(torch.uint8)[:, width:] = 0x7f
    return codes


def bound(av, bv, k, out):
    """Of each element: f32 sums of 128 exact products and of the scaled blocks, then the store's rounding.  A sum
    of n terms is off by at most n 2^-24 of the sum of magnitudes; the tensor cores may cut an addend where
    others round, which doubles it."""
    terms = 2 * (128 + 3 * (k // 128 + 1))
    e = (av.abs() @ bv.abs().t()) * terms * 2.0 ** -24
    return e + (out.abs() + e) * 2.0 ** -8 + 2.0 ** -133          # half a unit of 8 significant bits


PRODUCTS = [(1, 1, 1), (1, 130, 1000), (2, 128, 128), (3, 3584, 512), (7, 256, 7168), (16, 100, 272), (17, 384, 640), (33, 300, 129),
            (64, 512, 1024), (65, 256, 2048), (100, 1000, 300), (128, 256, 384), (129, 257, 255), (200, 2048, 640), (300, 130, 2000),
            (515, 770, 520), (1500, 520, 260)]


@pytest.mark.parametrize("layout", [ops.FP8_BLOCKS, ops.FP8_ROWS])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, layout):
    a, b = normal(m + 1, m, k).cuda(), normal(n + 2, n, k, scale=0.02).cuda()
    b[:, ::3] *= 4
    qa, sa = fp8.quantize_rows(a)
    qb, sb = (fp8.quantize_rows if layout == ops.FP8_ROWS else fp8.quantize_blocks)(b)
    av = R.values(qa[:, :k].cpu(), sa.cpu(), 1)
    bv = R.values(qb[:, :k].cpu(), sb.cpu(), 1 if layout == ops.FP8_ROWS else R.BLOCK)
    want = av @ bv.t()
    qa, qb = dirty(qa, k), dirty(qb, k)
    out = torch.full((m + 1, n), 7.0, dtype=BF16, device="cuda")
    assert ops.k3_moe_fp8_product(out, qa, sa, qb, sb, m, n, k, layout, ops.FP8_BF16, 0)
    assert bool(((out[:m].cpu().double() - want).abs() <= bound(av, bv, k, want)).all())
    assert bool((out[m] == 7).all())                                        # nothing past the end
    acc = normal(5, m, n, dtype=F32).cuda()
    before = acc.cpu().double()
    assert ops.k3_moe_fp8_product(acc, qa, sa, qb, sb, m, n, k, layout, ops.FP8_F32, 1)
    off = (acc.cpu().double() - before - want).abs()
    assert bool((off <= bound(av, bv, k, torch.zeros_like(want)) + (before.abs() + want.abs()) * 2.0 ** -23).all())
    plain = torch.empty_like(acc)
    assert ops.k3_moe_fp8_product(plain, qa, sa, qb, sb, m, n, k, layout, ops.FP8_F32, 0)
    assert bool(((plain.cpu().double() - want).abs() <= bound(av, bv, k, torch.zeros_like(want)) + want.abs() * 2.0 ** -23).all())


@pytest.mark.parametrize("layout", [ops.FP8_BLOCKS, ops.FP8_ROWS])
@pytest.mark.parametrize("m,n,k", [(2500, 2100, 2050), (700, 4000, 3000)])
def test_product_of_more_items_than_sms(m, n, k, layout):
    """Whole items for every SM, and the ones that are left split along the depth."""
    a, b = normal(m + 1, m, k).cuda(), normal(n + 2, n, k, scale=0.02).cuda()
    qa, sa = fp8.quantize_rows(a)
    qb, sb = (fp8.quantize_rows if layout == ops.FP8_ROWS else fp8.quantize_blocks)(b)
    av = R.values(qa[:, :k].cpu(), sa.cpu()[:, :-(-k // 128)], 1)
    bv = R.values(qb[:, :k].cpu(), sb.cpu()[:, :-(-k // 128)], 1 if layout == ops.FP8_ROWS else R.BLOCK)
    want = av @ bv.t()
    out = torch.empty(m, n, device="cuda")
    assert ops.k3_moe_fp8_product(out, dirty(qa, k), sa, dirty(qb, k), sb, m, n, k, layout, ops.FP8_F32, 0)
    assert bool(((out.cpu().double() - want).abs() <= bound(av, bv, k, torch.zeros_like(want)) + want.abs() * 2.0 ** -23).all())


@pytest.mark.parametrize("m", [1, 40, 300])
def test_product_of_large_and_small_scales(m):
    """Blocks 2^60 apart: each is scaled on its own."""
    n, k = 200, 640
    a, b = normal(1, m, k).float(), normal(2, n, k).float()
    a[:, 128:256] *= 2.0 ** 60
    a[:, 256:384] *= 2.0 ** -60
    b[:, 128:256] *= 2.0 ** -60
    b[:, 256:384] *= 2.0 ** 60
    qa, sa = fp8.quantize_rows(a.cuda())
    qb, sb = fp8.quantize_blocks(b.cuda())
    av, bv = R.values(qa.cpu(), sa.cpu(), 1), R.values(qb.cpu(), sb.cpu(), R.BLOCK)
    out = torch.empty(m, n, dtype=BF16, device="cuda")
    assert ops.k3_moe_fp8_product(out, qa, sa, qb, sb, m, n, k, ops.FP8_BLOCKS, ops.FP8_BF16, 0)
    want = av @ bv.t()
    assert bool(((out.cpu().double() - want).abs() <= bound(av, bv, k, want)).all())


@pytest.mark.parametrize("m", [3, 40, 300])
def test_a_row_that_is_not_finite_stays_alone(m):
    n, k = 300, 512
    a, b = normal(1, m, k).cuda(), normal(2, n, k).cuda()
    lin = fp8.Fp8Linear(*fp8.quantize_blocks(b), n, k)
    clean = lin.forward(a)
    a[1, 77] = float("inf")
    a[m - 1, 400] = float("nan")
    got = lin.forward(a)
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[m - 1]).all())
    keep = [i for i in range(m) if i not in (1, m - 1)]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("tokens,rows,columns", [(1, 256, 512), (5, 130, 1000), (70, 512, 300), (300, 384, 640)])
def test_linear_and_its_gradients(tokens, rows, columns):
    x, dy = normal(1, tokens, columns).cuda(), normal(2, tokens, rows, scale=1e-3).cuda()
    table, scales = fp8.quantize_blocks(normal(3, rows, columns, scale=0.02).cuda())
    w = R.values(table[:, :columns].cpu(), scales.cpu(), R.BLOCK)
    xv = R.values(*R.quantize(x.cpu(), 1), 1)
    dyv = R.values(*R.quantize(dy.cpu(), 1), 1)
    y = fp8.Fp8Linear(table, scales, rows, columns).forward(x)
    assert bool(((y.cpu().double() - xv @ w.t()).abs() <= bound(xv, w, columns, xv @ w.t())).all())
    grad = fp8.Fp8LinearGradient(*fp8.transpose_blocks(table, scales, rows, columns), rows, columns)
    dx = grad.by_input(dy)
    assert bool(((dx.cpu().double() - dyv @ w).abs() <= bound(dyv, w.t(), rows, dyv @ w)).all())
    dyt, xt = R.values(*R.quantize(dy.cpu().t(), 1), 1), R.values(*R.quantize(x.cpu().t(), 1), 1)
    want = dyt @ xt.t()
    dw = grad.by_weight(dy, x)
    limit = bound(dyt, xt, tokens, torch.zeros_like(want)) + want.abs() * 2.0 ** -23
    assert bool(((dw.cpu().double() - want).abs() <= limit).all())
    again = grad.by_weight(dy, x, into=dw.clone())
    assert bool(((again.cpu().double() - 2 * want).abs() <= 2 * limit + want.abs() * 2.0 ** -22).all())
    # against differences of the loss <dy, y> along a direction, the products' 8-bit operands aside: a code is off by
    # at most 2^-4 of its value, independently, so a sum of n terms by 2^-4 of the root of its terms' squares (x 4)
    dx_dir, dw_dir = normal(7, tokens, columns).double(), normal(8, rows, columns).double()
    loss = lambda xx, ww: float((dy.cpu().double() * (xx @ ww.t())).sum())  # noqa: E731
    x64 = x.cpu().double()
    by_x = loss(x64 + dx_dir, w) - loss(x64, w)                             # the loss is linear in each
    by_w = loss(x64, w + dw_dir) - loss(x64, w)
    noise = lambda p, q, d: 4 * 2.0 ** -4 * float(((p ** 2) @ (q ** 2) * d ** 2).sum().sqrt()) * 2 ** 0.5  # noqa: E731
    assert abs(float((dx.cpu().double() * dx_dir).sum()) - by_x) <= noise(dy.cpu().double(), w, dx_dir)
    assert abs(float((dw.cpu().double() * dw_dir).sum()) - by_w) <= noise(dy.cpu().double().t(), x64, dw_dir)


@pytest.mark.parametrize("start", [0, 1])
@pytest.mark.parametrize("tokens,rows,columns", [(1, 1, 1), (1, 3584, 7168), (2, 130, 1001), (15, 300, 640), (16, 2048, 136), (17, 129, 1000),
                                                 (33, 512, 2048), (63, 260, 131), (64, 7168, 2048)])
def test_linear_of_few_tokens(tokens, rows, columns, start):
    """Tokens quantised inside the product; `start`: from a place between 16-byte boundaries."""
    x = normal(tokens, tokens * columns + 1).cuda()[start:][:tokens * columns].view(tokens, columns)
    x[:, ::7] *= 50
    table, scales = fp8.quantize_blocks(normal(3, rows, columns, scale=0.02).cuda())
    dirty(table, columns)
    w = R.values(table.view(torch.uint8)[:, :columns].cpu().view(E4M3), scales.cpu(), R.BLOCK)
    xv = R.values(*R.quantize(x.cpu(), 1), 1)
    lin = fp8.Fp8Linear(table, scales, rows, columns)
    y = lin.forward(x)
    assert bool(((y.cpu().double() - xv @ w.t()).abs() <= bound(xv, w, columns, xv @ w.t())).all())
    assert torch.equal(y, lin.forward(x))


def expert_tables(seed, experts, hidden, expert_hidden):
    made = []
    for i, (r, c) in enumerate(((expert_hidden, hidden), (expert_hidden, hidden), (hidden, expert_hidden))):
        per = [fp8.quantize_blocks(normal(seed + 10 * i + e, r, c, scale=1.5 * c ** -0.5).cuda()) for e in range(experts)]
        made.append((torch.stack([p[0] for p in per]), torch.stack([p[1] for p in per])))
    return made


def expert_layer(tables, top_k, kind):
    return fp8.Fp8Experts(*tables[0], *tables[1], *tables[2], top_k=top_k, activation=kind)


def routes(seed, tokens, experts, top_k):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(tokens, experts, generator=g).topk(top_k, 1).indices.to(torch.int32)
    return ids, torch.rand(tokens, top_k, generator=g) + 0.1


def rel(got, want):
    return float((got.cpu().double() - want).norm() / want.norm())


# The rows' and the sum's rounding to bf16 (each 2^-8 of a value at most and 1.7e-3 of the norm: 2.4e-3 together)
# and the few codes of the activation on whose sides f32 and f64 sums fall (a part in 1e4, each 2^-4: 6e-4).
EXPERTS_REL = 3.5e-3


@pytest.mark.parametrize("kind", ["swiglu", "situ"])
@pytest.mark.parametrize("tokens,hidden,expert_hidden,experts,top_k", [
    (1, 512, 256, 8, 2), (1, 1024, 1040, 4, 4), (1, 128, 16, 33, 32), (1, 7168, 2048, 3, 3), (1, 16, 400, 1, 1), (1, 2064, 144, 20, 11), (2, 144, 80, 3, 1), (7, 256, 128, 16, 5), (33, 640, 384, 6, 3), (64, 528, 272, 5, 2),
    (150, 512, 256, 4, 4), (300, 400, 144, 33, 8), (700, 256, 384, 2, 2), (1200, 272, 160, 3, 1)])
def test_experts(tokens, hidden, expert_hidden, experts, top_k, kind):
    tables = expert_tables(tokens, experts, hidden, expert_hidden)
    x = normal(tokens + 1, tokens, hidden)
    ids, weights = routes(tokens + 2, tokens, experts, top_k)
    layer = expert_layer(tables, top_k, kind)
    out = layer.forward(x.cuda(), ids.cuda(), weights.cuda())
    cpu = [(c[..., :w].cpu(), s.cpu()) for (c, s), w in zip(tables, (hidden, hidden, expert_hidden))]
    want = R.experts(x, ids, weights, cpu, kind)
    assert rel(out, want) <= EXPERTS_REL
    assert torch.equal(out, layer.forward(x.cuda(), ids.cuda(), weights.cuda()))        # the same bits again
    shared = normal(4, tokens, hidden).cuda()
    with_shared = layer.forward(x.cuda(), ids.cuda(), weights.cuda(), shared)
    assert rel(with_shared, want + shared.cpu().double()) <= EXPERTS_REL


def test_experts_that_nobody_and_everybody_selects():
    tables = expert_tables(5, 9, 256, 128)
    x = normal(6, 400, 256)
    ids = torch.full((400, 2), 8, dtype=torch.int32)
    ids[:, 1] = 3
    ids[7, 1] = 0
    weights = torch.rand(400, 2, generator=torch.Generator().manual_seed(1))
    cpu = [(c[..., :w].cpu(), s.cpu()) for (c, s), w in zip(tables, (256, 256, 128))]
    out = expert_layer(tables, 2, "swiglu").forward(x.cuda(), ids.cuda(), weights.cuda())
    assert rel(out, R.experts(x, ids, weights, cpu, "swiglu")) <= EXPERTS_REL


@pytest.mark.parametrize("tokens", [1, 5, 200])
def test_an_id_that_is_no_expert_contributes_nothing(tokens):
    tables = expert_tables(5, 4, 256, 128)
    x = normal(6, tokens, 256).cuda()
    ids, weights = routes(2, tokens, 4, 3)
    ids[0, 1] = -1
    ids[tokens - 1, 2] = 4
    layer = expert_layer(tables, 3, "swiglu")
    layer.forward(normal(8, tokens, 256).cuda(), *(t.cuda() for t in routes(3, tokens, 4, 3)))      # what a call before leaves
    out = layer.forward(x, ids.cuda(), weights.cuda())
    assert ops.k3_moe_device_status() & 2
    assert ops.k3_moe_device_status_clear() and ops.k3_moe_device_status() == 0
    cpu = [(c[..., :w].cpu(), s.cpu()) for (c, s), w in zip(tables, (256, 256, 128))]
    assert rel(out, R.experts(x.cpu(), ids, weights, cpu, "swiglu")) <= EXPERTS_REL


def test_a_token_that_is_not_finite_stays_alone():
    tables = expert_tables(5, 4, 256, 128)
    x = normal(6, 50, 256).cuda()
    ids, weights = (t.cuda() for t in routes(2, 50, 4, 2))
    layer = expert_layer(tables, 2, "situ")
    clean = layer.forward(x, ids, weights)
    x[13, 200] = float("nan")
    got = layer.forward(x, ids, weights)
    assert bool(torch.isnan(got[13]).all())
    keep = [i for i in range(50) if i != 13]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("tokens", [1, 40, 600])
def test_tables_of_more_than_four_gigabytes(tokens):
    """The last expert of a large table gives the bits that it gives alone."""
    experts, hidden, expert_hidden = 300, 7168, 2048
    g = torch.Generator(device="cuda").manual_seed(3)
    tables = []
    for r, c in ((expert_hidden, hidden), (expert_hidden, hidden), (hidden, expert_hidden)):
        codes = torch.empty(experts, r, c, dtype=torch.uint8, device="cuda").random_(0, 256, generator=g)
        codes[-1] &= 0xf7                                                   # no NaN codes (0x7f, 0xff)
        scales = torch.rand(experts, -(-r // 128), -(-c // 128), generator=g, device="cuda") * 1e-4
        tables.append((codes.view(E4M3), scales))
    assert tables[0][0].numel() > 1 << 32
    x = normal(6, tokens, hidden).cuda()
    weights = torch.rand(tokens, 1, generator=g, device="cuda")
    last = torch.full((tokens, 1), experts - 1, dtype=torch.int32, device="cuda")
    got = expert_layer(tables, 1, "situ").forward(x, last, weights)
    # alone, among as many experts that nobody selects as the choice of kernel (by rows per expert) wants
    alone = [(torch.cat([c[-1:]] * 16), torch.cat([s[-1:]] * 16)) for c, s in tables]
    want = expert_layer(alone, 1, "situ").forward(x, torch.full_like(last, 15), weights)
    assert bool(torch.isfinite(want).all()) and torch.equal(got, want)


def test_another_stream_and_a_captured_call():
    tables = expert_tables(5, 4, 256, 128)
    layer = expert_layer(tables, 2, "swiglu")
    x = normal(6, 50, 256).cuda()
    ids, weights = (t.cuda() for t in routes(2, 50, 4, 2))
    want = layer.forward(x, ids, weights)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(layer.forward(x, ids, weights), want)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.forward(x, ids, weights)
    for seed in (1, 2):
        x.copy_(normal(seed, 50, 256))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer.forward(x, ids, weights))


def test_no_tokens():
    table, scales = fp8.quantize_blocks(normal(3, 64, 128).cuda())
    grad = fp8.Fp8LinearGradient(*fp8.transpose_blocks(table, scales, 64, 128), 64, 128)
    none = lambda n: torch.empty(0, n, dtype=BF16, device="cuda")           # noqa: E731
    assert fp8.Fp8Linear(table, scales, 64, 128).forward(none(128)).shape == (0, 64)
    assert not grad.by_weight(none(64), none(128)).any()
    assert fp8.quantize_rows(none(128))[0].shape == (0, 128)
    layer = expert_layer(expert_tables(5, 4, 256, 128), 2, "swiglu")
    empty = torch.empty(0, 2, device="cuda")
    assert layer.forward(none(256), empty.int(), empty).shape == (0, 256)
