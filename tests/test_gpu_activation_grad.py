"""Gradient of the gated activation with the routing weights, against 64 bits.

The exponentials and reciprocals are within some 2^-20 of their results (more for large gates, where the result is smaller by
more); 1e-5 of the magnitudes that are added covers them.  A bf16 output adds 2^-8 of the value."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import grouped, ops        # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
BETA, LINEAR = 4.0, 25.0


def parts(kind, g, u):
    """left, its derivative and the magnitudes behind it, right, its derivative; f64."""
    sig, rest = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    if kind == "swiglu":
        return g * sig, sig + g * sig * rest, sig + (g * sig * rest).abs(), u, torch.ones_like(u)
    left = BETA * torch.tanh(g / BETA) * sig
    first = sig / torch.cosh(g / BETA) ** 2
    return left, first + left * rest, first + (left * rest).abs(), LINEAR * torch.tanh(u / LINEAR), 1 / torch.cosh(u / LINEAR) ** 2


def reference(kind, d, gate, up, w):
    d, g, u, w = d.double(), gate.double(), up.double(), w.double().unsqueeze(1)
    left, d_left, size, right, d_right = parts(kind, g, u)
    values = {"d_gate": w * d * right * d_left, "d_up": w * d * left * d_right, "scaled": w * left * right,
              "d_weights": (d * left * right).sum(1)}
    sizes = {"d_gate": (w * d * right).abs() * size, "d_up": (w * d * left * d_right).abs(), "scaled": (w * left * right).abs(),
             "d_weights": (d * left * right).abs().sum(1)}
    return values, sizes


def check(name, got, want, size, terms=1):
    half = 2.0 ** -8 if got.dtype is BF16 else 2.0 ** -24
    err, bound = (got.double() - want).abs(), half * want.abs() + (1e-5 + terms * 2.0 ** -24) * size + 1e-36
    assert bool((err <= bound).all()), (name, float((err - bound).max()), float(err.max()))


def inputs(seed, rows, columns, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda s: (torch.randn(rows, columns, generator=g, device="cuda") * s).to(BF16)  # noqa: E731
    return normal(1e-2), normal(spread), normal(spread)


@pytest.mark.parametrize("kind", ["swiglu", "situ"])
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 2048), (3, 8), (16, 264), (77, 1023), (1183, 33), (1184, 40), (1300, 2056), (2000, 7)])
def test_against_64_bits(kind, rows, columns):
    d, gate, up = inputs(rows + columns, rows, columns)
    g = torch.Generator(device="cuda").manual_seed(rows)
    weights = torch.rand(rows, generator=g, device="cuda") * 3
    routes = torch.randperm(rows, generator=g, device="cuda").to(torch.int32)
    call = grouped.GatedActivation(kind, BETA, LINEAR)
    for w, r in ((weights, routes), (weights.view(1, -1), None), (None, None)):
        d_gate, d_up, scaled, d_weights = call.backward(d, gate, up, w, r)
        index = torch.arange(rows, device="cuda") if r is None else r.long()
        of_row = torch.ones(rows, device="cuda") if w is None else w.reshape(-1)[index]
        want, size = reference(kind, d, gate, up, of_row)
        for name, got in (("d_gate", d_gate), ("d_up", d_up), ("scaled", scaled)):
            check(name, got, want[name], size[name])
        assert d_weights.shape == ((rows,) if w is None else w.shape)
        check("d_weights", d_weights.reshape(-1)[index], want["d_weights"], size["d_weights"], columns)


@pytest.mark.parametrize("kind", ["swiglu", "situ"])
def test_large_and_small_gates(kind):
    """Every bf16 gate from -90 to 90 or so, where sigmoids and tanhs saturate and derivatives keep only what is left."""
    gate = torch.arange(0, 0x42b5, 7, device="cuda", dtype=torch.int32)
    gate = torch.cat([gate, gate | 0x8000]).to(torch.int16).view(BF16).view(1, -1).contiguous()
    up = torch.full_like(gate, 1.5)
    d = torch.ones_like(gate)
    d_gate, d_up, scaled, _ = grouped.GatedActivation(kind, BETA, LINEAR).backward(d, gate, up)
    want, size = reference(kind, d, gate, up, torch.ones(1, device="cuda"))
    for name, got in (("d_gate", d_gate), ("d_up", d_up), ("scaled", scaled)):
        # the exponent's rounding, 1.4e-7 of its size, comes on top
        check(name, got, want[name], size[name] * (1 + 0.02 * gate.double().abs()))
    swapped = grouped.GatedActivation(kind, BETA, LINEAR).backward(d, up, gate)
    want, size = reference(kind, d, up, gate, torch.ones(1, device="cuda"))
    for name, got in (("d_gate", swapped[0]), ("d_up", swapped[1]), ("scaled", swapped[2])):
        check(name, got, want[name], size[name] * (1 + 0.02 * gate.double().abs()))


@pytest.mark.parametrize("kind", ["swiglu", "situ"])
def test_gradient_against_differences(kind):
    rows, columns, step = 5, 96, 1e-5
    d, gate, up = inputs(3, rows, columns)
    g = torch.Generator(device="cuda").manual_seed(4)
    weights = torch.rand(rows, generator=g, device="cuda") + 0.5
    d_gate, d_up, _, d_weights = grouped.GatedActivation(kind, BETA, LINEAR).backward(d, gate, up, weights)

    def value(x, y, w):
        left, _, _, right, _ = parts(kind, x, y)
        return (d.double() * w.unsqueeze(1) * left * right).sum()
    x, y, w = gate.double(), up.double(), weights.double()
    for got, at in ((d_gate, 0), (d_up, 1), (d_weights, 2)):
        for _ in range(3):
            args = [x, y, w]
            v = torch.randn(args[at].shape, generator=g, device="cuda", dtype=torch.float64)
            plus, minus = list(args), list(args)
            plus[at], minus[at] = args[at] + step * v, args[at] - step * v
            slope = float((value(*plus) - value(*minus)) / (2 * step))
            size = float((got.double() * v).abs().sum())
            assert abs(float((got.double() * v).sum()) - slope) <= (2.0 ** -8 if at < 2 else 2e-5) * size + 1e-8


@pytest.mark.parametrize("columns", [64, 33])
@pytest.mark.parametrize("rows", [40, 1300])
def test_rows_of_no_group_are_not_touched(rows, columns):
    d, gate, up = inputs(5, rows, columns)
    d[:3] = float("nan")
    gate[rows - 5:] = float("nan")
    weights = torch.rand(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    routes = torch.arange(rows, device="cuda", dtype=torch.int32).flip(0).contiguous()
    routes[rows - 5:] = 7                                                  # what no dispatch wrote
    offsets = torch.tensor([3, 3, 20, rows - 5], dtype=torch.int32, device="cuda")
    _, _, _, d_weights = grouped.GatedActivation().backward(d, gate, up, weights, routes, offsets)
    want, size = reference("swiglu", d, gate, up, weights[routes.long()])
    inside = torch.arange(3, rows - 5, device="cuda")
    check("d_weights", d_weights[routes[inside].long()], want["d_weights"][inside], size["d_weights"][inside], columns)
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[routes[inside].long()] = False
    assert not d_weights[rest].any()
    # the C call leaves what the rows' outputs hold
    out = [torch.full_like(d, 5.0) for _ in range(3)]
    assert ops.k3_moe_activation_backward(*out, None, d, gate, up, weights, routes, offsets, 3, rows, columns, rows, ops.ACT_SWIGLU, 1.0, 1.0)
    for t in out:
        assert bool((t[:3] == 5).all()) and bool((t[rows - 5:] == 5).all()) and bool(torch.isfinite(t).all())


def test_a_route_past_the_weights_has_weight_0():
    d, gate, up = inputs(6, 4, 16)
    weights = torch.ones(3, device="cuda")
    routes = torch.tensor([0, 3, 2, -1], dtype=torch.int32, device="cuda")
    d_gate, d_up, scaled, d_weights = grouped.GatedActivation().backward(d, gate, up, weights, routes)
    for t in (d_gate, d_up, scaled):
        assert not t[1].any() and not t[3].any() and t[0].any() and t[2].any()
    assert float(d_weights[1]) == 0.0 and float(d_weights[0]) != 0.0 and float(d_weights[2]) != 0.0


@pytest.mark.parametrize("rows,columns", [(20, 264), (1300, 33)])
def test_in_place(rows, columns):
    d, gate, up = inputs(7, rows, columns)
    want = grouped.GatedActivation("situ").backward(d, gate, up)
    assert ops.k3_moe_activation_backward(gate, up, d, None, d, gate, up, None, None, None, 0, rows, columns, rows, ops.ACT_SITU, 4.0, 25.0)
    assert torch.equal(gate, want[0]) and torch.equal(up, want[1]) and torch.equal(d, want[2])


def test_no_rows_and_no_columns():
    for shape in ((0, 8), (3, 0)):
        t = torch.empty(shape, dtype=BF16, device="cuda")
        d_gate, d_up, scaled, d_weights = grouped.GatedActivation().backward(t, t, t)
        assert d_gate.shape == d_up.shape == scaled.shape == shape and d_weights.shape == (shape[0],) and not d_weights.any()
        assert grouped.GatedActivation().forward(t, t).shape == shape


def test_forward_is_the_activation_operator():
    _, gate, up = inputs(8, 9, 40)
    out = torch.empty_like(gate)
    assert ops.k3_moe_activation_bf16(out, gate, up, gate.numel(), ops.ACT_SITU, 4.0, 25.0)
    assert torch.equal(grouped.GatedActivation("situ").forward(gate, up), out)
