"""Grouped products, the activation's gradient and the norm where an element's number passes 32 bits: the rows and matrices
behind the 2^32nd element, against 64 bits."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import fp8, grouped, norm        # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def free():
    yield
    torch.cuda.empty_cache()


def near(got, want, size, depth):
    err = (got.double() - want).abs()
    assert bool((err <= depth * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all()), float(err.max())


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=BF16)


@pytest.mark.parametrize("form", ["forward", "by_input"])
def test_rows(form):
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, narrow, wide = (1 << 21) + 77, 8, 2056                           # 4.3 G elements out
    x = normal(g, rows, narrow)
    w = normal(g, 2, wide, narrow) if form == "forward" else normal(g, 2, narrow, wide)
    offsets = torch.tensor([0, 1000, rows - 5], dtype=torch.int32, device="cuda")
    product = grouped.GroupedProduct(w)
    got = product.forward(x, offsets) if form == "forward" else product.by_input(x, offsets)
    assert got.numel() > 1 << 32
    for at in (0, 999, 1000, 1 << 20, (1 << 32) // wide, rows - 40):
        part = slice(at, min(at + 30, rows - 5))
        of = [0 if r < 1000 else 1 for r in range(part.start, part.stop)]
        m = torch.stack([w[i] for i in of]).double()
        if form == "forward":
            m = m.transpose(1, 2)
        a = x[part].double()
        near(got[part], torch.einsum("rk,rkn->rn", a, m), torch.einsum("rk,rkn->rn", a.abs(), m.abs()), narrow)


def test_rows_read():
    """The products' inputs behind the 2^32nd element."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rows, n, k = (1 << 20) + 513, 16, 4104
    x = torch.zeros(rows, k, dtype=BF16, device="cuda")
    at = (1 << 32) // k
    for part in (slice(0, 20), slice(at - 10, at + 10), slice(rows - 20, rows)):
        x[part] = normal(g, 20, k)
    assert x.numel() > 1 << 32
    w, dy = normal(g, 3, n, k), normal(g, rows, n)
    offsets = torch.tensor([0, 10, at, rows], dtype=torch.int32, device="cuda")
    got = grouped.GroupedProduct(w).forward(x, offsets)
    for part, group in ((slice(0, 10), 0), (slice(10, 20), 1), (slice(at - 10, at), 1), (slice(at, at + 10), 2), (slice(rows - 20, rows), 2)):
        a, b = x[part].double(), w[group].double().t()
        near(got[part], a @ b, a.abs() @ b.abs(), k)
    dw = grouped.GroupedWeightGradient(3, n, k).forward(dy, x, offsets)
    for group, parts in ((0, [slice(0, 10)]), (1, [slice(10, 20), slice(at - 10, at)]), (2, [slice(at, at + 10), slice(rows - 20, rows)])):
        want = sum(dy[p].double().t() @ x[p].double() for p in parts)
        size = sum(dy[p].double().abs().t() @ x[p].double().abs() for p in parts)
        near(dw[group], want, size, 64)                                    # zeros add nothing


@pytest.mark.parametrize("n,k", [(4096, 4096), (4095, 4097)])
def test_matrices(n, k):
    """The weight's gradient and the matrices that are read, 5 G elements."""
    g = torch.Generator(device="cuda").manual_seed(3)
    groups, rows = 300, 600
    x, dy = normal(g, rows, k), normal(g, rows, n)
    cuts = [2 * i for i in range(groups + 1)]
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    dw = grouped.GroupedWeightGradient(groups, n, k).forward(dy, x, offsets, dtype=BF16)
    assert dw.numel() > 1 << 32
    for e in (0, 255, 256, 299):
        a, b = dy[2 * e:2 * e + 2].double().t(), x[2 * e:2 * e + 2].double()
        near(dw[e], a @ b, a.abs() @ b.abs(), 2)
    product = grouped.GroupedProduct(dw)                                   # as the matrices of the next layer's products
    out, dx = product.forward(x, offsets, dtype=F32), product.by_input(dy, offsets, dtype=F32)
    for e in (0, 255, 256, 299):
        part = slice(2 * e, 2 * e + 2)
        near(out[part], x[part].double() @ dw[e].double().t(), x[part].double().abs() @ dw[e].double().abs().t(), k)
        near(dx[part], dy[part].double() @ dw[e].double(), dy[part].double().abs() @ dw[e].double().abs(), n)


def test_activation_gradient():
    g = torch.Generator(device="cuda").manual_seed(4)
    rows, columns = (1 << 21) + 9, 2056
    gate = normal(g, rows, columns)
    d_gate, d_up, scaled, d_weights = grouped.GatedActivation().backward(gate, gate, gate)
    assert gate.numel() > 1 << 32
    for at in (0, (1 << 32) // columns - 3, rows - 8):
        x = gate[at:at + 8].double()
        sig = torch.sigmoid(x)
        assert torch.allclose(d_gate[at:at + 8].double(), x * x * (sig + x * sig * (1 - sig)), rtol=2.0 ** -8, atol=1e-4)
        assert torch.allclose(d_up[at:at + 8].double(), x * x * sig, rtol=2.0 ** -8, atol=1e-4)
        assert torch.allclose(scaled[at:at + 8].double(), x * x * sig, rtol=2.0 ** -8, atol=1e-4)
        assert torch.allclose(d_weights[at:at + 8].double(), (x * x * x * sig).sum(1), rtol=1e-4, atol=1e-2)


@pytest.mark.parametrize("hidden", [8192, 8190])
def test_norm(hidden):
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = (1 << 32) // hidden + 20
    x = normal(g, rows, hidden)
    weight = normal(g, hidden)
    call = norm.RmsNorm(weight)
    r = call.forward(x, x, codes=True)
    dx, _ = call.backward(x, r.sum, r.rstd, x)
    for at in (0, rows - 30, rows - 8):
        h = 2 * x[at:at + 8].double()
        rstd = torch.rsqrt(h.square().mean(1, keepdim=True) + call.epsilon)
        y = h * rstd * weight.double()
        assert torch.equal(r.sum[at:at + 8].double(), h)
        assert torch.allclose(r.y[at:at + 8].double(), y, rtol=1.01 * 2.0 ** -8, atol=0)
        full = r.scales[at:at + 8, :fp8.blocks(hidden)].double().repeat_interleave(128, 1)[:, :hidden]
        assert bool(((r.codes[at:at + 8, :hidden].double() * full - y).abs() <= 1.01 * 2.0 ** -4 * y.abs() + 2.0 ** -10 * full).all())
        gw, z = x[at:at + 8].double() * weight.double(), h * rstd
        want = h / 2 + rstd * (gw - z * (gw * z).mean(1, keepdim=True))
        assert torch.allclose(dx[at:at + 8].double(), want, rtol=2.0 ** -8, atol=1e-3)
