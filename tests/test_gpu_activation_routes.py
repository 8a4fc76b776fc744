"""The gated activation's gradient where routes have no row: past the routing weights, or doubled."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import grouped        # noqa: E402

BF16, I32 = torch.bfloat16, torch.int32


def fill_free_memory(elements):
    """Memory of that size which outputs are then made in holds NaN."""
    held = [torch.full((elements,), float("nan"), device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("routes", [[0, 5, 2, -1], [3, 3, 3, 0], [7, 8, 9, 10], [1, 2, 2, 2]])
@pytest.mark.parametrize("shape", [(4,), (2, 2)])
def test_weights_without_a_row_have_no_gradient(routes, shape):
    g = torch.Generator(device="cuda").manual_seed(1)
    d, gate, up = (torch.randn(4, 24, generator=g, device="cuda").to(BF16) for _ in range(3))
    weights = torch.ones(shape, device="cuda")
    for _ in range(3):
        fill_free_memory(4)
        _, _, _, d_weights = grouped.GatedActivation().backward(d, gate, up, weights, torch.tensor(routes, dtype=I32, device="cuda"))
        assert d_weights.shape == shape
        flat = d_weights.reshape(-1)
        for route in range(4):
            assert bool(flat[route] != 0) == (route in routes) and bool(torch.isfinite(flat[route]))
