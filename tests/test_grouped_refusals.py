"""What the grouped products, the activation's gradient and the norm refuse, before any launch: the C entry points by their
arguments, the Python forms by shapes, types and places."""
import pytest
import torch

from moonshine_b200 import build, fp8, grouped, norm, ops

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
CUDA0 = torch.device("cuda", 0)
P = 0x1000          # never dereferenced: every call below fails validation first


@pytest.fixture(scope="module")
def lib():
    from moonshine_b200 import _native
    build.build()
    return _native.lib()


def refuses(fn, good, bad):
    for at, value in bad:
        args = list(good)
        args[at] = value
        assert fn(*args) is False, (fn.__name__, at, value)


@pytest.mark.parametrize("name", ["k3_moe_grouped_product", "k3_moe_grouped_by_input", "k3_moe_grouped_by_weight"])
def test_grouped_products(lib, name):
    need = lib.k3_moe_grouped_workspace_bytes(40, 3)
    assert need > 0
    for rows, groups in ((0, 3), (40, 0), (40, 1025), ((1 << 30) + 1, 3)):
        assert lib.k3_moe_grouped_workspace_bytes(rows, groups) == 0
    assert lib.k3_moe_grouped_workspace_bytes(1 << 30, 1024) > lib.k3_moe_grouped_workspace_bytes(1 << 20, 1024) >= need
    # out, a, b, offsets, rows, groups, n, k, out type, accumulate, workspace, bytes, stream
    good = [P, P, P, P, 40, 3, 64, 64, 0, 0, P, need, None]
    refuses(getattr(lib, name), good,
            ((0, None), (1, None), (2, None), (3, None), (10, None), (4, 0), (5, 0), (5, 1025), (6, 0), (7, 0), (8, 2), (8, -1), (9, 1),
             (11, need - 1), (10, P + 8), (0, P + 1), (1, P + 1), (2, P + 1), (3, P + 2), (4, (1 << 30) + 1), (6, (1 << 30) + 1),
             (7, (1 << 30) + 1)))
    f32 = list(good)
    f32[8], f32[0] = 1, P + 2                                              # f32 between its words
    assert getattr(lib, name)(*f32) is False


def test_sizes_past_what_a_launch_takes(lib):
    need = lib.k3_moe_grouped_workspace_bytes(1 << 20, 1024)
    for n in (1 << 30, (1 << 30) - 1):                                     # the tensor-core kernels, the others
        assert lib.k3_moe_grouped_by_weight(P, P, P, P, 1 << 20, 1024, n, 1 << 20, 0, 0, P, need, None) is False


def test_activation_gradient(lib):
    # d_gate, d_up, scaled, d_weights, d_out, gate, up, weights, routes, offsets, groups, rows, columns, routes, kind, beta, linear, stream
    good = [P, P, P, P, P, P, P, P, P, P, 3, 4, 64, 4, 0, 4.0, 25.0, None]
    refuses(lib.k3_moe_activation_backward, good,
            ((0, None), (1, None), (4, None), (5, None), (6, None), (11, 0), (12, 0), (14, 2), (14, -1), (15, 0.0), (16, -1.0), (15, float("nan")),
             (0, P + 1), (1, P + 1), (2, P + 1), (4, P + 1), (5, P + 1), (6, P + 1), (3, P + 2), (7, P + 2), (8, P + 1), (9, P + 2),
             (11, (1 << 30) + 1), (12, (1 << 30) + 1)))


def test_norm(lib):
    # sum, y, codes, scales, rstd, x, residual, weight, rows, hidden, type, epsilon, stream
    good = [P, P, P, P, P, P, P, P, 4, 64, 0, 1e-5, None]
    refuses(lib.k3_moe_norm, good,
            ((5, None), (7, None), (2, None), (3, None), (8, 0), (9, 0), (9, 16385), (10, 2), (10, -1), (11, 0.0), (11, -1.0), (11, float("nan")),
             (0, P + 1), (1, P + 1), (2, P + 8), (3, P + 4), (4, P + 2), (5, P + 1), (6, P + 1), (7, P + 1), (8, (1 << 30) + 1)))
    nothing = list(good)
    nothing[1] = nothing[2] = nothing[3] = None
    assert lib.k3_moe_norm(*nothing) is False
    f32 = list(good)
    f32[10], f32[5] = 1, P + 2
    assert lib.k3_moe_norm(*f32) is False


def test_norm_gradient(lib):
    need = lib.k3_moe_norm_workspace_bytes(4, 64)
    assert need > 0 and lib.k3_moe_norm_workspace_bytes(0, 64) == lib.k3_moe_norm_workspace_bytes(4, 0) == 0
    assert lib.k3_moe_norm_workspace_bytes(4, 16385) == 0
    # dx, d_weight, dy, sum, rstd, d_sum, weight, rows, hidden, type, accumulate, workspace, bytes, stream
    good = [P, P, P, P, P, P, P, 4, 64, 0, 0, P, need, None]
    refuses(lib.k3_moe_norm_backward, good,
            ((0, None), (2, None), (3, None), (4, None), (6, None), (8, 0), (8, 16385), (9, 2), (11, None), (12, need - 1), (11, P + 8),
             (0, P + 1), (1, P + 2), (2, P + 1), (3, P + 1), (4, P + 2), (5, P + 1), (6, P + 1), (7, (1 << 30) + 1)))


# ------------------------------------------------------------------------------------------- the Python forms
class Placed:
    """What the checks look at of a tensor on a GPU."""
    def __init__(self, *shape, dtype=BF16, device=CUDA0):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, device

    def get_device(self):
        return self.device.index if self.device.type == "cuda" else -1

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()


def host(t):
    return Placed(*t.shape, dtype=t.dtype, device=torch.device("cpu"))


def other(t):
    return Placed(*t.shape, dtype=t.dtype, device=torch.device("cuda", 1))


@pytest.fixture()
def no_launch(monkeypatch):
    monkeypatch.setattr(fp8, "_current_device", lambda: 0)
    for name in vars(ops).copy():
        if name.startswith(("k3_moe_grouped", "k3_moe_norm", "k3_moe_activation", "k3_moe_fp8")) and "workspace" not in name:
            monkeypatch.setattr(ops, name, lambda *a, name=name, **k: pytest.fail(name + " was called"))


def misplaced(call, good, names):
    """Each tensor of a call on the host and on another device, by its name."""
    for at, name in enumerate(names):
        for wrong, message in ((host, "got one on cpu"), (other, "got one on cuda:1")):
            args = list(good)
            args[at] = wrong(good[at])
            with pytest.raises(ValueError, match=f"{name}: expected a tensor on the current CUDA device, {message}"):
                call(*args)


def test_grouped_product_form(no_launch, monkeypatch):
    for w in (torch.zeros(3, 16, 24), torch.zeros(16, 24, dtype=BF16), torch.zeros(3, 16, 24, dtype=BF16).transpose(1, 2)):
        with pytest.raises(ValueError, match=r"w: expected contiguous bfloat16 \[groups, n, k\]"):
            grouped.GroupedProduct(w)
    product = grouped.GroupedProduct(torch.zeros(3, 16, 24, dtype=BF16))
    x, dy, offsets = Placed(5, 24), Placed(5, 16), Placed(4, dtype=I32)
    with pytest.raises(ValueError, match="x: on cuda:0, the tables are on cpu"):
        product.forward(x, offsets)
    with pytest.raises(ValueError, match="dy: on cuda:0, the tables are on cpu"):
        product.by_input(dy, offsets)
    monkeypatch.setattr(product, "_device", CUDA0)
    misplaced(product.forward, [x, offsets], ["x", "offsets"])
    misplaced(product.by_input, [dy, offsets], ["dy", "offsets"])
    misplaced(lambda out: product.forward(x, offsets, out=out), [Placed(5, 16)], ["out"])
    misplaced(lambda into: product.forward(x, offsets, into=into), [Placed(5, 16, dtype=F32)], ["into"])
    for bad in (Placed(5, 23), Placed(5, 24, dtype=F32), Placed(24)):
        with pytest.raises(ValueError, match=r"x: expected \[rows, 24\]"):
            product.forward(bad, offsets)
    with pytest.raises(ValueError, match=r"dy: expected \[rows, 16\]"):
        product.by_input(x, offsets)
    for bad in (Placed(3, dtype=I32), Placed(4, dtype=torch.int64), Placed(4, 1, dtype=I32)):
        with pytest.raises(ValueError, match=r"offsets: expected torch.int32 \[4\]"):
            product.forward(x, bad)
    with pytest.raises(ValueError, match="dtype: bfloat16 or float32"):
        product.forward(x, offsets, dtype=torch.float16)
    for bad in (Placed(4, 16), Placed(5, 16, dtype=torch.float16)):
        with pytest.raises(ValueError, match=r"out: expected bfloat16 or float32 \[5, 16\]"):
            product.forward(x, offsets, out=bad)
    for bad in (Placed(4, 16, dtype=F32), Placed(5, 16)):
        with pytest.raises(ValueError, match=r"into: expected torch.float32 \[5, 16\]"):
            product.forward(x, offsets, into=bad)
    with pytest.raises(ValueError, match="out and into: one of them"):
        product.forward(x, offsets, out=Placed(5, 16), into=Placed(5, 16, dtype=F32))


def test_grouped_weight_gradient_form(no_launch):
    gradient = grouped.GroupedWeightGradient(3, 16, 24)
    dy, x, offsets = Placed(5, 16), Placed(5, 24), Placed(4, dtype=I32)
    misplaced(gradient.forward, [dy, x, offsets], ["dy", "x", "offsets"])
    misplaced(lambda into: gradient.forward(dy, x, offsets, into=into), [Placed(3, 16, 24, dtype=F32)], ["into"])
    with pytest.raises(ValueError, match="dy and x: different numbers of rows"):
        gradient.forward(dy, Placed(6, 24), offsets)
    with pytest.raises(ValueError, match=r"into: expected torch.float32 \[3, 16, 24\]"):
        gradient.forward(dy, x, offsets, into=Placed(3, 24, 16, dtype=F32))
    with pytest.raises(ValueError, match=r"offsets: expected torch.int32 \[4\]"):
        gradient.forward(dy, x, Placed(5, dtype=I32))


def test_gated_activation_form(no_launch):
    with pytest.raises(ValueError, match="activation: 'swiglu' or 'situ'"):
        grouped.GatedActivation("gelu")
    act = grouped.GatedActivation()
    t = lambda *s, **k: Placed(*s, **k)  # noqa: E731
    good = [t(6, 8), t(6, 8), t(6, 8), t(2, 3, dtype=F32), t(6, dtype=I32), t(4, dtype=I32)]
    misplaced(act.backward, good, ["d_out", "gate", "up", "weights", "routes", "offsets"])
    misplaced(act.forward, good[:2], ["gate", "up"])
    for at, bad, message in ((0, t(6, 8, dtype=F32), "d_out: expected"), (1, t(6, 9), r"gate: expected torch.bfloat16 \[6, 8\]"),
                             (2, t(5, 8), r"up: expected torch.bfloat16 \[6, 8\]"), (3, t(2, 3), "weights: expected float32"),
                             (4, t(5, dtype=I32), r"routes: expected torch.int32 \[6\]"), (4, t(6, dtype=torch.int64), "routes: "),
                             (5, t(1, dtype=I32), r"offsets: expected int32 \[groups \+ 1\]"), (5, t(4, dtype=F32), "offsets: ")):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError, match=message):
            act.backward(*args)
    with pytest.raises(ValueError, match="weights: expected float32, one for each of 6 rows or with routes"):
        act.backward(*good[:3], t(2, 4, dtype=F32))


def test_norm_form(no_launch, monkeypatch):
    for w in (torch.zeros(8), torch.zeros(8, 1, dtype=BF16), torch.zeros(16, dtype=BF16)[::2]):
        with pytest.raises(ValueError, match=r"weight: expected contiguous bfloat16 \[hidden\]"):
            norm.RmsNorm(w)
    call = norm.RmsNorm(torch.zeros(8, dtype=BF16))
    with pytest.raises(ValueError, match="x: on cuda:0, the tables are on cpu"):
        call.forward(Placed(3, 8))
    monkeypatch.setattr(call, "_device", CUDA0)
    misplaced(call.forward, [Placed(3, 8), Placed(3, 8)], ["x", "residual"])
    back = [Placed(3, 8), Placed(3, 8, dtype=F32), Placed(3, dtype=F32), Placed(3, 8, dtype=F32), Placed(8, dtype=F32)]
    misplaced(call.backward, back, ["dy", "sum", "rstd", "d_sum", "into"])
    with pytest.raises(ValueError, match=r"x: expected \[rows, 8\]"):
        call.forward(Placed(3, 9))
    with pytest.raises(ValueError, match=r"residual: expected torch.bfloat16 \[3, 8\]"):
        call.forward(Placed(3, 8), Placed(3, 8, dtype=F32))
    with pytest.raises(ValueError, match="y and codes: one of them at least"):
        call.forward(Placed(3, 8), y=False)
    for at, bad, message in ((0, Placed(3, 8, dtype=F32), r"dy: expected torch.bfloat16 \[3, 8\]"), (1, Placed(3, 7), r"sum: expected \[rows, 8\]"),
                             (2, Placed(4, dtype=F32), r"rstd: expected torch.float32 \[3\]"), (3, Placed(3, 8), r"d_sum: expected torch.float32 \[3, 8\]"),
                             (4, Placed(7, dtype=F32), r"into: expected torch.float32 \[8\]")):
        args = list(back)
        args[at] = bad
        with pytest.raises(ValueError, match=message):
            call.backward(*args)


def test_linear_of_codes(no_launch, monkeypatch):
    linear = fp8.Fp8Linear(torch.zeros(64, 128, dtype=torch.float8_e4m3fn), torch.ones(1, 1), 64, 128)
    codes, scales = Placed(3, 128, dtype=torch.float8_e4m3fn), Placed(3, 4, dtype=F32)
    with pytest.raises(ValueError, match="codes: on cuda:0, the tables are on cpu"):
        linear.forward_codes(codes, scales)
    monkeypatch.setattr(linear, "_device", CUDA0)
    misplaced(linear.forward_codes, [codes, scales], ["codes", "scales"])
    with pytest.raises(ValueError, match=r"scales: expected \[rows, 4\]"):
        linear.forward_codes(codes, Placed(3, 1, dtype=F32))
