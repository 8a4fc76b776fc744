"""E4M3 codes of the norm of bf16 rows: y / scale is 448 s w / max |s w| of the block, a quotient of numbers that 64 bits hold
exactly, so every code has to be the rounding of it, ties to the even one."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import fp8, norm, ops        # noqa: E402

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
HIDDEN = [1, 8, 127, 136, 257, 512, 1000, 1024, 1032, 2045, 2048, 3583, 4096, 4104, 7001, 7168, 8200, 16384]


def quotients(s, weight):
    """448 s w / max |s w| over each 128 columns, in 64 bits."""
    rows, hidden = s.shape
    p = torch.nn.functional.pad(s.double() * weight.double(), (0, -hidden % 128)).view(rows, -1, 128)
    largest = p.abs().amax(2, keepdim=True)
    return torch.where(largest > 0, 448 * p / largest.clamp(min=1e-300), 0.0).view(rows, -1)[:, :hidden]


def inputs(kind, rows, hidden):
    g = torch.Generator(device="cuda").manual_seed(rows + hidden)
    if kind == "normal":
        return torch.randn(rows, hidden, generator=g, device="cuda").to(BF16), (1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(BF16)
    # few values, so that many quotients are the middle between two codes
    x = torch.randint(-7, 8, (rows, hidden), generator=g, device="cuda").to(BF16)
    x[:, ::128] = 7                                                # of a block: 448 s w / (7 x 2) = 32 s w
    return x, (torch.randint(4, 9, (hidden,), generator=g, device="cuda") / 4).to(BF16)


@pytest.mark.parametrize("hidden", HIDDEN)
@pytest.mark.parametrize("rows", [1, 500])
@pytest.mark.parametrize("kind", ["normal", "few"])
@pytest.mark.parametrize("with_y", [False, True])
def test_every_code(hidden, rows, kind, with_y):
    x, weight = inputs(kind, rows, hidden)
    if kind == "few":
        weight[::128] = 2
    residual = torch.zeros_like(x) if rows > 1 else None
    x[rows // 2, hidden // 2:] = 0                                  # blocks of zeros
    r = norm.RmsNorm(weight).forward(x, residual, y=with_y, codes=True)
    q = quotients(x, weight).float()
    want = q.to(E4M3)
    if kind == "few" and hidden * rows > 1000:
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
        assert int(((q / step).frac().abs() == 0.5).sum()) > hidden * rows // 100      # ties are among them
    assert torch.equal(r.codes[:, :hidden].float(), want.float())
    assert ops.k3_moe_device_status() == 0


@pytest.mark.parametrize("hidden", [7168, 1000, 2045])
def test_products_near_the_ends_of_the_range(hidden):
    """Where s w leaves f32's range or comes near its ends, while y does not."""
    rows = 12
    x, weight = inputs("normal", rows, hidden)
    x[1] *= 2.0 ** -100
    x[2] *= 2.0 ** 55
    x[3] *= 2.0 ** -126
    x[4, :hidden // 2] *= 2.0 ** -120
    x[5] = 0
    x[6, 3:] = 0
    for exponent in (0, 75, -75, -100):
        w = (weight.double() * 2.0 ** exponent).to(BF16)
        r = norm.RmsNorm(w, 1e-5).forward(x, y=True, codes=True)
        h = x.double()
        y = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * w.double()
        full = r.scales[:, :fp8.blocks(hidden)].double().repeat_interleave(128, 1)[:, :hidden]
        assert torch.isfinite(r.y.float()).all() and torch.isfinite(full).all()
        err = (r.codes[:, :hidden].double() * full - y).abs()
        # half a code's step of the value or of the smallest steps, and f32's smallest numbers
        assert bool((err <= (2.0 ** -4 + 2.0 ** -16) * y.abs() + 2.0 ** -10 * full + 2.0 ** -140).all()), exponent
